// Dropout from a counter-based generator; the mask is a function of (seed, offset, element index)
// and is never stored, so the backward pass regenerates it.
//
// Element e = row * cols + col (whatever the strides) takes word e % 4 of block e / 4 of
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011)
// with key = seed and counter = (block, offset). It is kept iff its word >= floor(p 2^32), and a
// kept element is x / (1 - p): out = kept ? x * (1 / (1 - p)) : 0, plus residual where given. A
// dropped element is 0 whatever x holds (NaN and infinity included).
//
// HBM bound once the generator is out of the way: 16384 x 4096 bf16 with a residual (403 MB) 75 us,
// 5.4 TB/s; with the round keys added up per thread and one run per thread it took 91 us.
#include <cmath>

#include "features.cuh"

namespace gpb {

// The ten round keys are the same for every thread: the host adds them up once, and each round is
// two wide multiplies and two three-way xors with a constant-bank operand. The generator is what a
// plain dropout's arithmetic consists of: 20 wide multiplies per four elements.
struct DropoutArgs {
  const void* x;
  const void* res;
  void* out;
  int64_t x_ld, res_ld, out_ld;
  int64_t rows, cols, count;
  uint64_t offset;
  uint32_t key[20];
  uint32_t border;
  float scale;
};

__device__ __forceinline__ uint4 philox(uint64_t block, const DropoutArgs& A) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)A.offset, c3 = (uint32_t)(A.offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ A.key[2 * r];
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ A.key[2 * r + 1];
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}

// RUNS aligned runs of VEC elements per thread, a block's width apart (VEC a multiple of 4: VEC / 4
// generator blocks each); all their loads are issued before the first generator round. FLAT: every
// operand is contiguous, so the element index is the address; otherwise VEC divides cols and a run
// stays inside one row.
template <typename T, int VEC, int RUNS, bool FLAT>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const __grid_constant__ DropoutArgs A) {
  const int64_t run0 = (int64_t)blockIdx.x * (256 * RUNS) + threadIdx.x;
  Pack<T, VEC> x[RUNS], res[RUNS];
  int64_t oi[RUNS];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int64_t e = (run0 + u * 256) * VEC;
    if (e >= A.count) break;
    int64_t xi = e, ri = e;
    oi[u] = e;
    if constexpr (!FLAT) {
      const int64_t row = e / A.cols, col = e - row * A.cols;
      xi = row * A.x_ld + col;
      ri = row * A.res_ld + col;
      oi[u] = row * A.out_ld + col;
    }
    x[u] = *reinterpret_cast<const Pack<T, VEC>*>((const T*)A.x + xi);
    if (A.res) res[u] = *reinterpret_cast<const Pack<T, VEC>*>((const T*)A.res + ri);
  }
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int64_t e = (run0 + u * 256) * VEC;
    if (e >= A.count) break;
    float v[VEC];
#pragma unroll
    for (int b = 0; b < VEC / 4; ++b) {
      const uint4 w = philox((uint64_t)(e / 4 + b), A);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float kept = ws[q] >= A.border ? to_f(x[u].v[4 * b + q]) * A.scale : 0.f;
        v[4 * b + q] = A.res ? kept + to_f(res[u].v[4 * b + q]) : kept;
      }
    }
    store_vec<T, VEC>((T*)A.out + oi[u], v);
  }
}

// Any strides, widths and alignments: one thread per generator block, element by element.
template <typename T>
__global__ void __launch_bounds__(256) dropout_any_kernel(const __grid_constant__ DropoutArgs A) {
  const int64_t block = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (block * 4 >= A.count) return;
  const uint4 w = philox((uint64_t)block, A);
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t e = block * 4 + q;
    if (e >= A.count) break;
    const int64_t row = e / A.cols, col = e - row * A.cols;
    float v = to_f(((const T*)A.x)[row * A.x_ld + col]);
    v = ws[q] >= A.border ? v * A.scale : 0.f;
    if (A.res) v += to_f(((const T*)A.res)[row * A.res_ld + col]);
    ((T*)A.out)[row * A.out_ld + col] = from_f<T>(v);
  }
}

template <typename T>
static int dropout_launch(const DropoutArgs& A, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const bool flat = A.x_ld == A.cols && A.out_ld == A.cols && (!A.res || A.res_ld == A.cols);
  const bool ptrs = aligned16(A.x) && aligned16(A.out) && (!A.res || aligned16(A.res));
  const bool rows_ok = A.cols % VEC == 0 && A.x_ld % VEC == 0 && A.out_ld % VEC == 0 &&
                       (!A.res || A.res_ld % VEC == 0);
  // Two runs per thread once that still gives every SM its threads.
  const bool two = A.count / VEC >= (int64_t)kFeatSMs * 4096;
  const unsigned g1 = (unsigned)ceil_div(A.count / VEC, 256), g2 = (unsigned)ceil_div(A.count / VEC, 512);
  if (ptrs && flat && A.count % VEC == 0) {
    if (two)
      dropout_vec_kernel<T, VEC, 2, true><<<g2, 256, 0, st>>>(A);
    else
      dropout_vec_kernel<T, VEC, 1, true><<<g1, 256, 0, st>>>(A);
  } else if (ptrs && rows_ok) {
    if (two)
      dropout_vec_kernel<T, VEC, 2, false><<<g2, 256, 0, st>>>(A);
    else
      dropout_vec_kernel<T, VEC, 1, false><<<g1, 256, 0, st>>>(A);
  } else {
    dropout_any_kernel<T><<<(unsigned)ceil_div(ceil_div(A.count, 4), 256), 256, 0, st>>>(A);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

}  // namespace gpb

using namespace gpb;

extern "C" int gpb_dropout(int32_t device, void* stream, int32_t dtype, int64_t rows, int64_t cols,
                           void* out_dev, int64_t out_ld, const void* x_dev, int64_t x_ld,
                           const void* residual_dev, int64_t residual_ld, double p, uint64_t seed,
                           uint64_t offset) {
  clear_error();
  GPB_REQUIRE(dtype_ok(dtype), GPB_ERR_INVALID, "unknown element type %d", dtype);
  GPB_REQUIRE(rows >= 0 && cols >= 0, GPB_ERR_INVALID, "negative size");
  GPB_REQUIRE(p >= 0.0 && p < 1.0, GPB_ERR_INVALID, "dropout probability must be in [0, 1), got %g",
              p);
  if (rows == 0 || cols == 0) return GPB_OK;
  const int es = dtype_bytes(dtype);
  GPB_REQUIRE(cols <= ((int64_t)1 << 38) / rows, GPB_ERR_INVALID, "%lld x %lld elements are too many",
              (long long)rows, (long long)cols);
  GPB_REQUIRE(out_dev && x_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(out_ld >= cols && x_ld >= cols && (!residual_dev || residual_ld >= cols),
              GPB_ERR_INVALID, "leading dimension below the %lld columns", (long long)cols);
  GPB_REQUIRE(elem_aligned(out_dev, es) && elem_aligned(x_dev, es) && elem_aligned(residual_dev, es),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const Extent out = block_extent(out_dev, rows, cols, out_ld, es);
  GPB_REQUIRE((out_dev == x_dev && out_ld == x_ld) ||
                  !overlaps(out, block_extent(x_dev, rows, cols, x_ld, es)),
              GPB_ERR_INVALID, "out overlaps x (in place needs the same pointer and stride)");
  GPB_REQUIRE((out_dev == residual_dev && out_ld == residual_ld) ||
                  !overlaps(out, block_extent(residual_dev, rows, cols, residual_ld, es)),
              GPB_ERR_INVALID, "out overlaps residual (in place needs the same pointer and stride)");
  GPB_DEVICE_SCOPE(device);
  DropoutArgs A{};
  A.x = x_dev;
  A.res = residual_dev;
  A.out = out_dev;
  A.x_ld = x_ld;
  A.res_ld = residual_ld;
  A.out_ld = out_ld;
  A.rows = rows;
  A.cols = cols;
  A.count = rows * cols;
  A.offset = offset;
  for (int r = 0; r < 10; ++r) {
    A.key[2 * r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
    A.key[2 * r + 1] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
  }
  A.border = (uint32_t)std::floor(p * 4294967296.0);
  A.scale = (float)(1.0 / (1.0 - p));
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case GPB_DTYPE_F32: return dropout_launch<float>(A, st);
    case GPB_DTYPE_F16: return dropout_launch<__half>(A, st);
    default: return dropout_launch<__nv_bfloat16>(A, st);
  }
}
