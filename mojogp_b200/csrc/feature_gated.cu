// Gated projection unit: both projections, the activation and the product in one kernel.
//   gate = x Wg' + bg,  up = x Wu' + bu,  out = act(gate) * up
// x [rows][inner], Wg and Wu [outer][inner], row-major; out [rows][outer].
// Backward, with gate and up recomputed (they are never stored):
//   dgate = dout up act'(gate),  dup = dout act(gate)
//   dx = dgate Wg + dup Wu,  dWg = dgate' x,  dWu = dup' x,  dbg, dbu = column sums
//
// A few rows (few_rows) read every weight once for a handful of multiply-adds: HBM bound, on the CUDA
// cores in fp32 (gated_rows_*; 1 row, 2048 -> 8192 bf16, 67 MB: 16 us). More rows run on the tensor cores
// (gated_gemm.cuh), up to some 200 of them for the time of the weights' reading.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "gated_gemm.cuh"

namespace gpb {

constexpr int kFewRows = 8;

// Set by a kernel whose bounded wait ran out; read and cleared by gpb_feature_status.
__device__ int g_feature_err;

struct GatedArgs {
  const void* x;
  const void* wg;
  const void* wu;
  const void* bg;
  const void* bu;
  const void* dout;
  void* out;  // forward
  int64_t x_ld, w_ld, out_ld, dout_ld;
  int64_t rows, inner, outer;
  int32_t act;
};

struct GatedGrads {
  void* dx;
  int64_t dx_ld;
  void* dwg;
  void* dwu;
  int64_t dw_ld;
  void* dbg;
  void* dbu;
};

// ------------------------------------------------------------- few rows
// A weight vector, read once: past L1, which keeps x.
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}
template <typename T>
__device__ __forceinline__ T load_once(const T* p) {
  return *p;
}
// A vector's elements as pairs: 16 bytes, or one element and a zero.
template <typename T, int P>
__device__ __forceinline__ void to_pairs(const uint4& q, float2 (&o)[P]) {
  unpack16(q, o, (const T*)nullptr);
}
template <typename T, int P>
__device__ __forceinline__ void to_pairs(const T& q, float2 (&o)[P]) {
  o[0] = make_float2(to_f(q), 0.f);
}

// One warp (WPO = 1) or one block (WPO = 8) per output column; lanes run along the weight row. BACK
// writes dgate and dup [rows][outer] in fp32. HBM bound: a lane issues U vectors of each weight row
// before it uses the first.
template <typename T, int ROWS, int VEC, int WPO, bool BACK>
__global__ void __launch_bounds__(256) gated_rows_kernel(const GatedArgs A, float* dg, float* du) {
  using Raw = typename std::conditional<VEC == 1, T, uint4>::type;
  constexpr int P = VEC == 1 ? 1 : VEC / 2, U = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = WPO == 1 ? (int64_t)blockIdx.x * 8 + warp : (int64_t)blockIdx.x;
  float2 g2[ROWS], u2[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) g2[m] = u2[m] = make_float2(0.f, 0.f);
  if (n < A.outer) {
    const T* wg = (const T*)A.wg + n * A.w_ld;
    const T* wu = (const T*)A.wu + n * A.w_ld;
    constexpr int kStep = (WPO == 1 ? 32 : 256) * VEC;
    for (int k0 = (WPO == 1 ? lane : (int)threadIdx.x) * VEC; k0 < A.inner; k0 += U * kStep) {
      Raw a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * kStep;
        if (k < A.inner) {
          a[u] = load_once((const Raw*)(wg + k));
          b[u] = load_once((const Raw*)(wu + k));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * kStep;
        if (k < A.inner) {
          float2 p[P], q[P];
          to_pairs<T>(a[u], p);
          to_pairs<T>(b[u], q);
#pragma unroll
          for (int m = 0; m < ROWS; ++m) {
            if (m < A.rows) {
              float2 x[P];
              to_pairs<T>(*(const Raw*)((const T*)A.x + m * A.x_ld + k), x);
#pragma unroll
              for (int i = 0; i < P; ++i) {
                g2[m] = __ffma2_rn(x[i], p[i], g2[m]);
                u2[m] = __ffma2_rn(x[i], q[i], u2[m]);
              }
            }
          }
        }
      }
    }
  }
  float g[ROWS], u[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    g[m] = g2[m].x + g2[m].y;
    u[m] = u2[m].x + u2[m].y;
    for (int o = 16; o > 0; o >>= 1) {
      g[m] += __shfl_xor_sync(0xffffffffu, g[m], o);
      u[m] += __shfl_xor_sync(0xffffffffu, u[m], o);
    }
  }
  if constexpr (WPO == 8) {
    __shared__ float sums[8][2][ROWS];
    if (lane == 0)
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        sums[warp][0][m] = g[m];
        sums[warp][1][m] = u[m];
      }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      g[m] = u[m] = 0.f;
      for (int w = 0; w < 8; ++w) {
        g[m] += sums[w][0][m];
        u[m] += sums[w][1][m];
      }
    }
  }
  if (n >= A.outer || (WPO == 8 && warp > 0)) return;
  float gate = g[0], up = u[0];  // lane m finishes row m
#pragma unroll
  for (int m = 1; m < ROWS; ++m)
    if (lane == m) {
      gate = g[m];
      up = u[m];
    }
  if (lane < ROWS && lane < A.rows) {
    if (A.bg) gate += to_f(((const T*)A.bg)[n]);
    if (A.bu) up += to_f(((const T*)A.bu)[n]);
    const float z[1] = {gate};
    float value[1], slope[1];
    gated_act<BACK>(A.act, z, value, slope);
    if constexpr (BACK) {
      const float dy = to_f(((const T*)A.dout)[lane * A.dout_ld + n]);
      dg[lane * A.outer + n] = dy * up * slope[0];
      du[lane * A.outer + n] = dy * value[0];
    } else {
      ((T*)A.out)[lane * A.out_ld + n] = from_f<T>(value[0] * up);
    }
  }
}

// dx of few rows: a thread owns VEC columns of the weights and walks a range of their rows
// (blockIdx.y); the ranges' sums are joined by gated_rows_join_kernel.
template <typename T, int ROWS, int VEC>
__global__ void __launch_bounds__(128) gated_rows_dx_kernel(const GatedArgs A, const float* dg,
                                                            const float* du, int64_t per,
                                                            float* partial) {
  const int64_t k = ((int64_t)blockIdx.x * 128 + threadIdx.x) * VEC;
  if (k >= A.inner) return;
  const int64_t n0 = blockIdx.y * per, n1 = n0 + per < A.outer ? n0 + per : A.outer;
  float acc[ROWS][VEC];
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[m][i] = 0.f;
#pragma unroll 4
  for (int64_t n = n0; n < n1; ++n) {
    float a[VEC], b[VEC];
    load_vec<T, VEC>((const T*)A.wg + n * A.w_ld + k, a);
    load_vec<T, VEC>((const T*)A.wu + n * A.w_ld + k, b);
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      if (m < A.rows) {
        const float p = dg[m * A.outer + n], q = du[m * A.outer + n];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[m][i] = fmaf(p, a[i], fmaf(q, b[i], acc[m][i]));
      }
    }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
    if (m < A.rows)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        partial[((int64_t)blockIdx.y * A.rows + m) * A.inner + k + i] = acc[m][i];
}

// dWg, dWu and the bias gradients of few rows: sums of ROWS outer products, written once.
template <typename T, int ROWS, int VEC>
__global__ void __launch_bounds__(128) gated_rows_dw_kernel(const GatedArgs A, const GatedGrads G,
                                                            const float* dg, const float* du) {
  const int64_t k = ((int64_t)blockIdx.y * 128 + threadIdx.x) * VEC;
  const int64_t n = blockIdx.x;
  float p[ROWS], q[ROWS], sp = 0.f, sq = 0.f;
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    p[m] = m < A.rows ? dg[m * A.outer + n] : 0.f;
    q[m] = m < A.rows ? du[m * A.outer + n] : 0.f;
    sp += p[m];
    sq += q[m];
  }
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    if (G.dbg) ((T*)G.dbg)[n] = from_f<T>(sp);
    if (G.dbu) ((T*)G.dbu)[n] = from_f<T>(sq);
  }
  if (k >= A.inner) return;
  float a[VEC], b[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = b[i] = 0.f;
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    if (m < A.rows) {
      float x[VEC];
      load_vec<T, VEC>((const T*)A.x + m * A.x_ld + k, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        a[i] = fmaf(p[m], x[i], a[i]);
        b[i] = fmaf(q[m], x[i], b[i]);
      }
    }
  }
  if (G.dwg) store_vec<T, VEC>((T*)G.dwg + n * G.dw_ld + k, a);
  if (G.dwu) store_vec<T, VEC>((T*)G.dwu + n * G.dw_ld + k, b);
}

// ------------------------------------------------------------- helpers
// dx of few rows: the sum of the ranges' partial sums [range][M][N], 32 elements per block, 32 threads
// along the ranges of each.
template <typename T>
__global__ void __launch_bounds__(1024) gated_rows_join_kernel(const float* __restrict__ partial,
                                                               int ranges, int64_t M, int64_t N, T* c,
                                                               int64_t c_ld) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (e < M * N)
#pragma unroll 4
    for (int r = part; r < ranges; r += 32) s += partial[r * M * N + e];
  sums[part][lane] = s;
  __syncthreads();
  float v = sums[lane][part];  // warp: element, lane: ranges
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t out = (int64_t)blockIdx.x * 32 + part;
  if (lane == 0 && out < M * N) c[(out / N) * c_ld + out % N] = from_f<T>(v);
}

// Matrices to tensor-core operands, one per blockIdx.y: fp32 weights to three bf16 planes, or a matrix
// whose rows are not 16-byte aligned to a copy whose are (`copy`). Columns up to ld are zeros.
struct PackArgs {
  const void* src[3];
  void* dst[3];
  int64_t rows[3], src_ld[3];
  int32_t copy[3];
  int64_t cols, ld;
};
// 16 bytes from an address that is only 2-byte aligned, of which the first `bytes` are asked for: the one or
// two aligned blocks that hold them, shifted.
__device__ __forceinline__ void load_blocks(const void* p, int64_t bytes, uint4& a, uint4& b) {
  const int off = (int)((uintptr_t)p & 15);
  const uint4* q = reinterpret_cast<const uint4*>((const char*)p - off);
  a = b = make_uint4(0, 0, 0, 0);
  if (bytes > 0) a = q[0];
  if (off + (bytes < 16 ? bytes : 16) > 16) b = q[1];
}
__device__ __forceinline__ uint4 shift_blocks(const void* p, const uint4& a, const uint4& b) {
  const int off = (int)((uintptr_t)p & 15);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t h[6], o[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) h[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) o[i] = off & 4 ? h[i + 1] : h[i];
  const int bits = (off & 2) * 8;
  return make_uint4(__funnelshift_r(o[0], o[1], bits), __funnelshift_r(o[1], o[2], bits),
                    __funnelshift_r(o[2], o[3], bits), __funnelshift_r(o[3], o[4], bits));
}

// HBM bound. A thread takes a few columns at a time (16 bits: eight, read as the aligned 16-byte blocks that
// hold them; fp32: two), and a block consecutive ones, rows end to end: whole lines whatever the rows' width
// and alignment, and no idle lanes at a row's end. Lanes assigned to rows, and unaligned words 16 or 32
// bytes apart, went through L1 several times: forward 94812 x 519 -> 51 bf16 126 us in all, 85 this way;
// 21764 x 3975 fp16 99 us of packing, now 62 (5.6 TB/s).
template <typename T>
struct PackShape {
  static constexpr int kCols = sizeof(T) == 4 ? 2 : 8;
  static constexpr int kItems = sizeof(T) == 4 ? 8 : 4;  // per thread
};
template <typename T, typename D>
__global__ void __launch_bounds__(256) gated_pack_kernel(const __grid_constant__ PackArgs A) {
  constexpr int COLS = PackShape<T>::kCols, ITEMS = PackShape<T>::kItems;
  const int o = blockIdx.y;
  const int64_t rows = A.rows[o], first = (int64_t)blockIdx.x * (256 * ITEMS);
  const uint32_t per = (uint32_t)(A.ld / COLS);
  const int64_t row0 = first / per;
  if (row0 >= rows) return;
  const uint32_t at0 = (uint32_t)(first - row0 * per) + threadIdx.x;
  const int left_rows = (int)(rows - row0 < (1 << 30) ? rows - row0 : 1 << 30);
  const T* src0 = (const T*)A.src[o] + row0 * A.src_ld[o];
  int r[ITEMS], c[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const uint32_t at = at0 + u * 256;
    r[u] = (int)(at / per);
    c[u] = (int)(at - r[u] * per) * COLS;
  }
  if constexpr (sizeof(T) == 4) {
    float2 w[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const T* src = src0 + r[u] * A.src_ld[o] + c[u];
      const bool in = r[u] < left_rows;
      w[u].x = in && c[u] < A.cols ? src[0] : 0.f;
      w[u].y = in && c[u] + 1 < A.cols ? src[1] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      if (r[u] >= left_rows) break;
      const int64_t at = (row0 + r[u]) * A.ld + c[u];
      if (A.copy[o]) {
        *reinterpret_cast<float2*>((T*)A.dst[o] + at) = w[u];
      } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<uint32_t*>((D*)A.dst[o] + k * rows * A.ld + at) = gg_part<D>(w[u]);
      }
    }
  } else {
    uint4 a[ITEMS], b[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u)
      load_blocks(src0 + r[u] * A.src_ld[o] + c[u], r[u] < left_rows ? 2 * (A.cols - c[u]) : 0, a[u],
                  b[u]);
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      if (r[u] >= left_rows) break;
      const uint4 q = shift_blocks(src0 + r[u] * A.src_ld[o] + c[u], a[u], b[u]);
      uint32_t h[4] = {q.x, q.y, q.z, q.w};
      const int64_t left = A.cols - c[u];
      if (left < COLS) {  // columns past the row are zeros
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * i + 1 >= left) h[i] = 2 * i < left ? h[i] & 0xFFFFu : 0u;
      }
      *reinterpret_cast<uint4*>((T*)A.dst[o] + (row0 + r[u]) * A.ld + c[u]) =
          make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
}

// Joins a projection's ranges and runs its epilogue: 32 rows x 32 columns to a block (blocks along the
// columns first), a warp to a row.
template <typename T, typename D, int PD, bool BACK>
__global__ void __launch_bounds__(1024) gated_finish_kernel(const __grid_constant__ GgArgs A) {
  __shared__ float sums[32][2][33];
  float scale = 1.f;  // of float16 factors
  if constexpr (kGgScaled<D> && BACK) {
    if (A.redo) {
      const int k = gg_factor_exp(*A.largest);
      if (k == 0) return;
      scale = gg_pow2(k);
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned across = (unsigned)((A.N + 31) / 32), by = blockIdx.x / across, bx = blockIdx.x - by * across;
  const int64_t n = (int64_t)bx * 32 + lane, ld = (A.N + 15) / 16 * 16;
  const bool in = n < A.N;
  const float bg = in && A.bg ? to_f(((const T*)A.bg)[n]) : 0.f;
  const float bu = in && A.bu ? to_f(((const T*)A.bu)[n]) : 0.f;
  float sg = 0.f, su = 0.f;
  const int64_t m = (int64_t)by * 32 + warp;
  if (m < A.M && in) {
    const float* src = A.partial + m * ld + n;
    float gate = 0.f, up = 0.f;
#pragma unroll 4
    for (int s = 0; s < A.splits; ++s) {
      gate += src[(2 * s) * A.M * ld];
      up += src[(2 * s + 1) * A.M * ld];
    }
    up += bu;
    const float z[1] = {gate + bg};
    float value[1], slope[1];
    gated_act<BACK>(A.act, z, value, slope);
    if constexpr (BACK) {
      const float dy = to_f(((const T*)A.dout)[m * A.dout_ld + n]);
      const float d[2] = {dy * up * slope[0], dy * value[0]};
      sg = d[0];
      su = d[1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float rest = d[h] * scale;
#pragma unroll
        for (int p = 0; p < PD; ++p) {
          const D part = from_f<D>(rest);
          ((D*)A.out[h])[p * A.plane + m * A.out_ld + n] = part;
          rest -= to_f(part);
        }
      }
    } else {
      ((T*)A.out[0])[m * A.out_ld + n] = from_f<T>(value[0] * up);
    }
  }
  if constexpr (BACK) {
    if constexpr (kGgScaled<D>) {
      const uint32_t top =
          __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(gg_magnitude(sg), gg_magnitude(su))));
      if (lane == 0 && !A.redo && top > 0) atomicMax(A.largest, top);
    }
    if (!A.col_sums) return;
    sums[warp][0][lane] = sg;
    sums[warp][1][lane] = su;
    __syncthreads();
    // Warp w adds column w's rows, one per lane.
    const int64_t c = (int64_t)bx * 32 + warp;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s = sums[lane][h][warp];
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0 && c < A.N) A.col_sums[((int64_t)by * 2 + h) * A.N + c] = s;
    }
  }
}

// The backward pass's joins in one launch: the ranges of dWg and dWu, then those of dx (in range order),
// then the column sums of dgate and dup (32 columns to a block, 32 threads along the partial rows).
struct RangeSums {
  const float* partial;  // [ranges][halves][M][N rounded up to 16]
  int64_t ranges, M, N, ld;
  int32_t halves;
  void* out[2];
  int64_t blocks;        // of 1024 elements
};
struct JoinArgs {
  RangeSums dw, dx;
  const float* col_sums;
  int64_t sum_rows, outer;
  void* db[2];
};
template <typename T>
__device__ __forceinline__ void range_join(const RangeSums& A, int64_t block) {
  const int64_t ld = (A.N + 15) / 16 * 16, one = A.M * ld;
  const int64_t e = block * 1024 + threadIdx.x;
  if (e >= A.halves * one) return;
  const int half = e >= one;
  const int64_t f = e - half * one, row = f / ld, col = f - row * ld;
  T* dst = (T*)A.out[half];
  if (!dst || col >= A.N) return;
  float s = 0.f;
#pragma unroll 4
  for (int64_t r = 0; r < A.ranges; ++r) s += A.partial[r * A.halves * one + e];
  dst[row * A.ld + col] = from_f<T>(s);
}
template <typename T>
__global__ void __launch_bounds__(1024) gated_join_kernel(const __grid_constant__ JoinArgs A) {
  if (blockIdx.x < A.dw.blocks)
    range_join<T>(A.dw, blockIdx.x);
  else if (blockIdx.x < A.dw.blocks + A.dx.blocks)
    range_join<T>(A.dx, blockIdx.x - A.dw.blocks);
  else
    column_join<T>(A.col_sums, A.sum_rows, A.outer, (T*)A.db[0], (T*)A.db[1],
                   blockIdx.x - A.dw.blocks - A.dx.blocks);
}

// ------------------------------------------------------------------ host
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int encode_fn(EncodeTiled* fn) {
  static std::atomic<EncodeTiled> cached{nullptr};
  *fn = cached.load(std::memory_order_acquire);
  if (!*fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    GPB_CHECK_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    GPB_REQUIRE(p && q == cudaDriverEntryPointSuccess, GPB_ERR_CUDA,
                "cuTensorMapEncodeTiled is not available");
    *fn = (EncodeTiled)p;
    cached.store(*fn, std::memory_order_release);
  }
  return GPB_OK;
}

// An operand as TMA reads it: `planes` matrices [rows][cols] of 16-bit elements, or one of fp32, whose
// rows are a multiple of 16 bytes apart.
struct Operand {
  const void* p = nullptr;
  bool f32 = false;
  int64_t rows = 0, cols = 0, ld = 0, plane = 0;
  int planes = 1;
};

static int make_map(const Operand& o, int box_cols, int box_rows, CUtensorMap* map) {
  EncodeTiled fn;
  GPB_TRY(encode_fn(&fn));
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const int64_t plane = o.planes > 1 ? o.plane : o.rows * o.ld;
  const int es = o.f32 ? 4 : 2;
  const cuuint64_t strides[2] = {(cuuint64_t)(o.ld * es), (cuuint64_t)(plane * es)};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  const CUresult r =
      fn(map, o.f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
         const_cast<void*>(o.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
         o.f32            ? CU_TENSOR_MAP_SWIZZLE_NONE
         : box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                          : CU_TENSOR_MAP_SWIZZLE_64B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  GPB_REQUIRE(r == CUDA_SUCCESS, GPB_ERR_CUDA, "tensor map of %lld x %lld (stride %lld): error %d",
              (long long)o.rows, (long long)o.cols, (long long)o.ld, (int)r);
  return GPB_OK;
}

// Workspace of a call; every offset from its 32-byte aligned base is a multiple of 256 bytes.
struct GatedPlan {
  bool few = false;                    // CUDA-core path
  int planes = 1;                      // of packed x and weights
  int planes_d = 1;                    // of dgate and dup
  int64_t ldk = 0, ldn = 0;            // leading dimensions of packed operands and of dgate / dup
  int64_t x = 0, wg = 0, wu = 0;       // packed operands
  int64_t dg = 0, du = 0, plane_d = 0; // dgate and dup (elements between planes)
  int64_t partial = 0, total = 0;
  int tile_n = 0;                      // GG_DW column tile
  int splits = 1, kb_per = 1;          // GG_DW
  int splits_p = 1, kb_per_p = 1;      // GG_PROJ
  int64_t partial_p = 0;
  int splits_x = 1, kb_per_x = 1;      // GG_DX
  int64_t partial_x = 0;
  int64_t sums = 0;                    // column sums of dgate and dup
  int64_t largest = 0;                 // float16: bits of the largest |dgate|, |dup|
  int ranges_x = 1;                    // dx of few rows
};

// The kernels store whole 32-byte sectors into the workspace (st.global.v8), while a caller's is 16-byte
// aligned: its base is rounded up, into 16 bytes that the size asked for has to spare.
static int64_t workspace_need(const GatedPlan& P) { return P.total > 0 ? P.total + 16 : 0; }
static char* workspace_base(void* p) { return (char*)(((uintptr_t)p + 31) & ~(uintptr_t)31); }

static int64_t take(int64_t& at, int64_t bytes) {
  const int64_t o = at;
  at += round_up(bytes, 256);
  return o;
}

// 16-bit dgate and dup are kept as two planes (16 and more significant bits) up to this many
// multiply-adds per product, as one above. One plane's rounding adds to the outputs' own: 1.4 times
// their error, and more where few terms or few outputs average it. The second plane doubles the MMAs
// of three of the four products (backward, bf16 silu with bias: 2048 x 256 -> 512 49 us against 48 with
// one plane, 4096 x 512 -> 512 55 against 47, 8192 x 512 -> 512 76 against 62). Above the bound it would
// cost half the call's time or more, and the outputs' sums are long enough to average the rounding.
constexpr int64_t kTwoPlanes = (int64_t)1 << 31;

// Stages of a 16-bit product's reduction that one accumulator takes. The tensor core truncates every term
// at 2^-25 of the accumulator, half of that on average, so k terms of one sign lose some k 2^-27: 16384 terms
// 2^-13, half of float16's own rounding (2^20 terms in one range came out 6e-3 short). Longer reductions
// split into ranges whose partial sums are added in fp32 (16 bytes an output for every 65536 operations).
static int64_t longest_range(int planes) { return 16384 / kGgBK / planes; }

// Rows of an A tile that a single row tile loads: whole groups of 8 (the swizzle's unit).
static int tile_rows(int64_t rows) {
  return rows < kGgBM ? (int)round_up(rows, 8) : kGgBM;
}
// Column tile of a GG_DX / GG_DW product with n output columns.
static int plain_tile(int64_t n, bool f32) { return n <= 64 ? 64 : n <= 128 || f32 ? 128 : 256; }
// MMA width of GG_PROJ: gate and up columns of one tile. The widest tile that its columns fill, or a
// narrower one where that finds more SMs: a tile's time goes with the 128 + nb rows that a stage loads
// (bf16, 16 rows, 2048 -> 8192: 64 tiles of 256 26 us, 128 tiles of 128 20 us).
static int proj_tile(int64_t rows, int64_t outer, bool f32) {
  int best = 64;
  int64_t least = INT64_MAX;
  for (int nb = outer <= 32 ? 64 : outer <= 64 || f32 ? 128 : 256; nb >= 64; nb /= 2) {
    const int64_t tiles = ceil_div(rows, kGgBM) * ceil_div(outer, nb / 2);
    const int64_t time = ceil_div(tiles, kFeatSMs) * (kGgBM + nb);
    if (time < least) {
      least = time;
      best = nb;
    }
  }
  return best;
}

// Rows up to which a call runs on the CUDA cores. Weights of a quarter million elements on: 16-bit, 2
// (2048 -> 8192 bf16 forward at 4 rows 39 us against 23.5 on the tensor cores, backward 105 against 75; at
// 2 rows 26.6 against 23.4, 72.6 against 74.5); fp32, whose tensor-core path packs the weights into
// planes first, all of kFewRows (57 us against 114, 181 against 212), but 4 where rows cannot be read as
// vectors (2047 -> 8191 at 8 rows 225 against 118, 427 against 247; at 4 rows 84 against 118). Smaller
// weights: launches decide, and this path has the fewer (501 -> 333 bf16 at 8 rows 11 us against 15,
// backward 28 against 48).
static int few_rows(int64_t inner, int64_t outer, bool f32) {
  if (inner * outer < (1 << 18)) return kFewRows;
  return !f32 ? 2 : inner % 4 ? 4 : kFewRows;
}

static GatedPlan gated_plan(int64_t rows, int64_t inner, int64_t outer, int32_t dtype, bool backward) {
  GatedPlan P;
  const bool f32 = dtype == GPB_DTYPE_F32;
  int64_t at = 0;
  if (rows <= few_rows(inner, outer, f32)) {
    P.few = true;
    if (!backward) return P;
    P.dg = take(at, rows * outer * 4);
    P.du = take(at, rows * outer * 4);
    const int vec = 16 / dtype_bytes(dtype);
    const int64_t cols = ceil_div(inner, 128 * vec);
    P.ranges_x = (int)std::max<int64_t>(
        1, std::min<int64_t>(ceil_div(outer, 16), ceil_div(4 * kFeatSMs, cols)));
    P.partial = take(at, P.ranges_x * rows * inner * 4);
    P.total = at;
    return P;
  }
  P.planes = f32 ? 3 : 1;
  P.ldk = round_up(inner, 8);
  P.ldn = round_up(outer, 16);
  P.x = take(at, rows * P.ldk * dtype_bytes(dtype));
  P.wg = take(at, P.planes * outer * P.ldk * 2);
  P.wu = take(at, P.planes * outer * P.ldk * 2);
  {
    // Few tiles split a projection's reduction, into ranges that outlast the further launch: 1024 deep,
    // 256 for fp32 (8192 -> 1024 bf16 at 16 rows: 44 us in one range, 23.5 in four).
    const int64_t kb = ceil_div(inner, f32 ? kGgSplitBK : kGgBK);
    const int64_t tiles = ceil_div(rows, kGgBM) * ceil_div(outer, proj_tile(rows, outer, f32) / 2);
    int64_t want = std::max<int64_t>(1, std::min<int64_t>(kFeatSMs / tiles, inner / (f32 ? 256 : 1024)));
    if (!f32) want = std::max(want, ceil_div(kb, longest_range(1)));
    P.kb_per_p = (int)ceil_div(kb, want);
    P.splits_p = (int)ceil_div(kb, P.kb_per_p);
    P.partial_p = take(at, P.splits_p > 1 ? P.splits_p * 2 * rows * round_up(outer, 16) * 4 : 0);
  }
  if (backward) {
    P.planes_d = f32 ? 3 : rows * inner * outer <= kTwoPlanes ? 2 : 1;
    P.plane_d = rows * P.ldn;
    P.dg = take(at, P.planes_d * P.plane_d * 2);
    P.du = take(at, P.planes_d * P.plane_d * 2);
    P.tile_n = plain_tile(inner, f32);
    const int64_t tiles = (outer <= 64 ? 1 : 2 * ceil_div(outer, kGgBM)) * ceil_div(inner, P.tile_n);
    const int bk = f32 ? kGgSplitBK : kGgBK;
    const int64_t kb = ceil_div(rows, bk);
    // At least 8 stages per range; as many ranges as fill the SMs twice.
    int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * kFeatSMs / tiles, kb / 8));
    if (!f32) want = std::max(want, ceil_div(kb, longest_range(P.planes_d)));
    P.kb_per = (int)ceil_div(kb, want);
    P.splits = (int)ceil_div(kb, P.kb_per);
    P.partial = take(at, P.splits > 1 ? P.splits * 2 * outer * round_up(inner, 16) * 4 : 0);
    // dx: the reduction is 2 outer long; ranges of at least 8 stages (4 of fp32's longer ones)
    // while they find idle SMs (bf16,
    // 16 rows, 2048 -> 8192: 8 tiles, 159 us in one range).
    const int64_t kbx = 2 * ceil_div(outer, kGgBK);
    const int64_t tiles_x = ceil_div(rows, kGgBM) * ceil_div(inner, P.tile_n);
    int64_t want_x = std::max<int64_t>(1, std::min<int64_t>(kFeatSMs / tiles_x, kbx / (f32 ? 4 : 8)));
    if (!f32) want_x = std::max(want_x, ceil_div(kbx, longest_range(P.planes_d)));
    P.kb_per_x = (int)ceil_div(kbx, want_x);
    P.splits_x = (int)ceil_div(kbx, P.kb_per_x);
    P.partial_x = take(at, P.splits_x > 1 ? P.splits_x * rows * round_up(inner, 16) * 4 : 0);
    P.sums = take(at, 4 * ceil_div(rows, kGgBM) * 2 * outer * 4);
    P.largest = take(at, dtype == GPB_DTYPE_F16 ? 4 : 0);
  }
  P.total = at;
  return P;
}

template <int MODE, int NB, int PA, int PB, typename T, typename D, int PD, bool BACK, int CTAS = 1>
static int gg_launch(const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0,
                     const CUtensorMap& b1, GgArgs G, cudaStream_t st) {
  using S = GgShape<MODE, NB, PA, PB, CTAS>;
  // CTA pairs once they still leave an item for every pair of SMs.
  if constexpr (CTAS == 1 && NB == 256 && PA == 1 && PB == 1) {
    if (G.tiles_m > 1 && ceil_div(G.tiles_m, 2) * (int64_t)G.tiles_n * G.splits >= kFeatSMs / 2)
      return gg_launch<MODE, NB, PA, PB, T, D, PD, BACK, 2>(a0, a1, b0, b1, G, st);
  }
  constexpr auto kernel = gated_gemm_kernel<MODE, NB, PA, PB, T, D, PD, BACK, CTAS>;
  GPB_TRY(allow_smem<kernel>(S::kSmem));
  void* err = nullptr;
  GPB_CHECK_CUDA(cudaGetSymbolAddress(&err, g_feature_err));
  G.err = (int*)err;
  G.idesc = gg_idesc(std::is_same<D, __nv_bfloat16>::value, MODE == GG_DW, MODE != GG_PROJ, NB,
                     CTAS * kGgBM);
  G.tiles_m = (int32_t)ceil_div(G.tiles_m, CTAS);
  const int64_t items = (int64_t)G.tiles_m * G.tiles_n * G.splits;
  const unsigned grid = CTAS * (unsigned)std::min<int64_t>(items, kFeatSMs / CTAS);
  kernel<<<grid, S::kThreads, S::kSmem, st>>>(a0, a1, b0, b1, G);
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

// Alignment of a matrix's rows: 2 = 32 bytes, 1 = 16 bytes, 0 = less.
static int row_align(const void* p, int64_t row_bytes) {
  const uint64_t bits = (uint64_t)(uintptr_t)p | (uint64_t)row_bytes;
  return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
}

// x and the weights as TMA reads them: where they lie when their rows are aligned, copied into the
// workspace otherwise; fp32 weights as planes (fp32 x is split inside the products).
template <typename T, typename D>
static int gated_operands(const GatedArgs& A, const GatedPlan& P, char* ws, Operand* x, Operand* wg,
                          Operand* wu, cudaStream_t st) {
  PackArgs K{};
  K.cols = A.inner;
  K.ld = P.ldk;
  int count = 0;
  int64_t most = 0;
  auto operand = [&](const void* p, int64_t rows, int64_t ld, char* packed, Operand* o, bool planes) {
    o->rows = rows;
    o->cols = A.inner;
    o->p = p;
    o->ld = ld;
    o->f32 = sizeof(T) == 4 && !planes;
    if (!planes && aligned16(p) && ld * sizeof(T) % 16 == 0) return;
    o->p = packed;
    o->ld = P.ldk;
    o->planes = planes ? P.planes : 1;
    o->plane = rows * P.ldk;
    K.src[count] = p;
    K.dst[count] = packed;
    K.rows[count] = rows;
    K.src_ld[count] = ld;
    K.copy[count] = !planes;
    most = std::max(most, rows);
    ++count;
  };
  constexpr bool kPlanes = sizeof(T) == 4;
  operand(A.x, A.rows, A.x_ld, ws + P.x, x, false);
  operand(A.wg, A.outer, A.w_ld, ws + P.wg, wg, kPlanes);
  operand(A.wu, A.outer, A.w_ld, ws + P.wu, wu, kPlanes);
  if (count) {
    using S = PackShape<T>;
    const int64_t blocks = ceil_div(most * P.ldk, (int64_t)S::kCols * 256 * S::kItems);
    gated_pack_kernel<T, D><<<dim3((unsigned)blocks, count), 256, 0, st>>>(K);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

template <typename T, typename D, int PL, int PD, bool BACK>
static int gated_project(const GatedArgs& A, const GatedPlan& P, char* ws, const Operand& x,
                         const Operand& wg, const Operand& wu, GgArgs G, cudaStream_t st) {
  const int nb = proj_tile(A.rows, A.outer, PL == 3);
  const int bn = nb / 2;
  CUtensorMap mx, mg, mu;
  constexpr int BK = PL == 3 ? kGgSplitBK : kGgBK;
  GPB_TRY(make_map(wg, BK, bn, &mg));
  GPB_TRY(make_map(wu, BK, bn, &mu));
  G.a_rows = tile_rows(A.rows);
  GPB_TRY(make_map(x, BK, G.a_rows, &mx));
  G.M = A.rows;
  G.N = A.outer;
  G.tiles_m = (int32_t)ceil_div(A.rows, kGgBM);
  G.tiles_n = (int32_t)ceil_div(A.outer, bn);
  G.kblocks = (int32_t)ceil_div(A.inner, BK);
  G.segs = 1;
  G.splits = P.splits_p;
  G.kb_per = P.kb_per_p;
  G.partial = (float*)(ws + P.partial_p);
  G.bg = A.bg;
  G.bu = A.bu;
  G.act = A.act;
  G.dout = A.dout;
  G.dout_ld = A.dout_ld;
  auto run = [&]() {
    switch (nb) {
      case 64: return gg_launch<GG_PROJ, 64, PL, PL, T, D, PD, BACK>(mx, mx, mg, mu, G, st);
      case 128: return gg_launch<GG_PROJ, 128, PL, PL, T, D, PD, BACK>(mx, mx, mg, mu, G, st);
      default:
        if constexpr (PL == 1)
          return gg_launch<GG_PROJ, 256, PL, PL, T, D, PD, BACK>(mx, mx, mg, mu, G, st);
        return (int)GPB_ERR_UNSUPPORTED;
    }
  };
  constexpr int passes = BACK && kGgScaled<D> ? 2 : 1;  // the second one scales, where it has to
  for (G.redo = 0; G.redo < passes; ++G.redo) {
    if (G.redo == 0 || G.splits == 1) GPB_TRY(run());
    if (G.splits > 1) {
      const unsigned grid = (unsigned)(ceil_div(A.outer, 32) * 4 * ceil_div(A.rows, kGgBM));
      gated_finish_kernel<T, D, PD, BACK><<<grid, 1024, 0, st>>>(G);
      GPB_CHECK_CUDA(cudaGetLastError());
    }
  }
  return GPB_OK;
}

template <int MODE, typename T, typename D, int PL, int PD>
static int gated_plain(const CUtensorMap& a0, const CUtensorMap& a1, const Operand& b0,
                       const Operand& b1, int nb, GgArgs& G, cudaStream_t st) {
  CUtensorMap m0, m1;
  constexpr int BK = gg_splits(MODE, PL) ? kGgSplitBK : kGgBK;
  GPB_TRY(make_map(b0, 64, BK, &m0));
  GPB_TRY(make_map(b1, 64, BK, &m1));
  switch (nb) {
    case 64: return gg_launch<MODE, 64, PD, PL, T, D, PD, false>(a0, a1, m0, m1, G, st);
    case 128: return gg_launch<MODE, 128, PD, PL, T, D, PD, false>(a0, a1, m0, m1, G, st);
    default:
      if constexpr (PL == 1)
        return gg_launch<MODE, 256, PD, PL, T, D, PD, false>(a0, a1, m0, m1, G, st);
      return GPB_ERR_UNSUPPORTED;
  }
}

template <typename T, int ROWS, int VEC, bool BACK>
static int gated_rows_launch(const GatedArgs& A, float* dg, float* du, cudaStream_t st) {
  // One warp per output column while that gives every SM 16 warps, else a block per column.
  if (A.outer >= 16 * kFeatSMs)
    gated_rows_kernel<T, ROWS, VEC, 1, BACK>
        <<<(unsigned)ceil_div(A.outer, 8), 256, 0, st>>>(A, dg, du);
  else
    gated_rows_kernel<T, ROWS, VEC, 8, BACK><<<(unsigned)A.outer, 256, 0, st>>>(A, dg, du);
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, int VEC, bool BACK>
static int gated_rows_pick(const GatedArgs& A, float* dg, float* du, cudaStream_t st) {
  if (A.rows <= 1) return gated_rows_launch<T, 1, VEC, BACK>(A, dg, du, st);
  if (A.rows <= 2) return gated_rows_launch<T, 2, VEC, BACK>(A, dg, du, st);
  if (A.rows <= 4) return gated_rows_launch<T, 4, VEC, BACK>(A, dg, du, st);
  return gated_rows_launch<T, kFewRows, VEC, BACK>(A, dg, du, st);
}

template <typename T, int ROWS, int VEC>
static int gated_rows_grads(const GatedArgs& A, const GatedGrads& G, const GatedPlan& P, float* dg,
                            float* du, float* partial, cudaStream_t st) {
  const int64_t cols = ceil_div(A.inner, 128 * VEC);
  if (G.dx) {
    const int64_t per = ceil_div(A.outer, P.ranges_x);
    const int ranges = (int)ceil_div(A.outer, per);
    gated_rows_dx_kernel<T, ROWS, VEC>
        <<<dim3((unsigned)cols, ranges), 128, 0, st>>>(A, dg, du, per, partial);
    GPB_CHECK_CUDA(cudaGetLastError());
    gated_rows_join_kernel<T><<<(unsigned)ceil_div(A.rows * A.inner, 32), 1024, 0, st>>>(
        partial, ranges, A.rows, A.inner, (T*)G.dx, G.dx_ld);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  if (G.dwg || G.dwu || G.dbg || G.dbu) {
    const unsigned gy = G.dwg || G.dwu ? (unsigned)cols : 1;
    gated_rows_dw_kernel<T, ROWS, VEC><<<dim3((unsigned)A.outer, gy), 128, 0, st>>>(A, G, dg, du);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

template <typename T, int VEC>
static int gated_rows_backward(const GatedArgs& A, const GatedGrads& G, const GatedPlan& P, char* ws,
                               cudaStream_t st) {
  float *dg = (float*)(ws + P.dg), *du = (float*)(ws + P.du), *partial = (float*)(ws + P.partial);
  GPB_TRY((gated_rows_pick<T, VEC, true>(A, dg, du, st)));
  if (A.rows <= 1) return gated_rows_grads<T, 1, VEC>(A, G, P, dg, du, partial, st);
  if (A.rows <= 2) return gated_rows_grads<T, 2, VEC>(A, G, P, dg, du, partial, st);
  if (A.rows <= 4) return gated_rows_grads<T, 4, VEC>(A, G, P, dg, du, partial, st);
  return gated_rows_grads<T, kFewRows, VEC>(A, G, P, dg, du, partial, st);
}

// x and weights readable as 16-byte vectors.
template <typename T>
static bool gated_vec(const GatedArgs& A) {
  constexpr int V = 16 / sizeof(T);
  return A.inner % V == 0 && A.x_ld % V == 0 && A.w_ld % V == 0 && aligned16(A.x) &&
         aligned16(A.wg) && aligned16(A.wu);
}

template <typename T, typename D, int PL>
static int gated_forward(const GatedArgs& A, char* ws, const GatedPlan& P, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (P.few)
    return gated_vec<T>(A) ? gated_rows_pick<T, V, false>(A, nullptr, nullptr, st)
                           : gated_rows_pick<T, 1, false>(A, nullptr, nullptr, st);
  Operand x, wg, wu;
  GPB_TRY((gated_operands<T, D>(A, P, ws, &x, &wg, &wu, st)));
  GgArgs G{};
  G.out[0] = A.out;
  G.out_ld = A.out_ld;
  G.vec = row_align(A.out, A.out_ld * sizeof(T));
  return gated_project<T, D, PL, PL, false>(A, P, ws, x, wg, wu, G, st);
}

template <typename T, typename D, int PL, int PD>
static int gated_backward_tc(const GatedArgs& A, const GatedGrads& R, char* ws, const GatedPlan& P,
                          cudaStream_t st) {
  Operand x, wg, wu;
  GPB_TRY((gated_operands<T, D>(A, P, ws, &x, &wg, &wu, st)));
  float* partial = (float*)(ws + P.partial);
  uint32_t* largest = (uint32_t*)(ws + P.largest);
  if constexpr (kGgScaled<D>) GPB_CHECK_CUDA(cudaMemsetAsync(largest, 0, sizeof(*largest), st));
  Operand dg, du;
  dg.p = ws + P.dg;
  du.p = ws + P.du;
  dg.rows = du.rows = A.rows;
  dg.cols = du.cols = A.outer;
  dg.ld = du.ld = P.ldn;
  dg.planes = du.planes = PD;
  dg.plane = du.plane = P.plane_d;
  {
    GgArgs G{};
    G.largest = largest;
    G.out[0] = ws + P.dg;
    G.out[1] = ws + P.du;
    G.out_ld = P.ldn;
    G.plane = P.plane_d;
    G.vec = row_align(A.dout, A.dout_ld * sizeof(T));
    if (R.dbg || R.dbu) G.col_sums = (float*)(ws + P.sums);
    GPB_TRY((gated_project<T, D, PL, PD, true>(A, P, ws, x, wg, wu, G, st)));
  }
  if (R.dx) {
    GgArgs G{};
    G.largest = largest;
    const int nb = plain_tile(A.inner, PL == 3);
    G.M = A.rows;
    G.N = A.inner;
    G.tiles_m = (int32_t)ceil_div(A.rows, kGgBM);
    G.tiles_n = (int32_t)ceil_div(A.inner, nb);
    G.kblocks = (int32_t)ceil_div(A.outer, kGgBK);
    G.segs = 2;
    G.splits = P.splits_x;
    G.kb_per = P.kb_per_x;
    G.partial = (float*)(ws + P.partial_x);
    G.out[0] = R.dx;
    G.out_ld = R.dx_ld;
    G.vec = row_align(R.dx, R.dx_ld * sizeof(T));
    CUtensorMap a0, a1;
    G.a_rows = tile_rows(A.rows);
    GPB_TRY(make_map(dg, kGgBK, G.a_rows, &a0));
    GPB_TRY(make_map(du, kGgBK, G.a_rows, &a1));
    GPB_TRY((gated_plain<GG_DX, T, D, PL, PD>(a0, a1, wg, wu, nb, G, st)));
  }
  if (R.dwg || R.dwu) {
    GgArgs G{};
    G.largest = largest;
    const bool joined = A.outer <= 64;
    G.M = A.outer;
    G.N = A.inner;
    G.half_tiles = joined ? 0 : (int32_t)ceil_div(A.outer, kGgBM);
    G.tiles_m = joined ? 1 : 2 * G.half_tiles;
    G.tiles_n = (int32_t)ceil_div(A.inner, P.tile_n);
    constexpr int BK = PL == 3 ? kGgSplitBK : kGgBK;
    G.kblocks = (int32_t)ceil_div(A.rows, BK);
    G.segs = 1;
    G.splits = P.splits;
    G.kb_per = P.kb_per;
    G.out[0] = R.dwg;
    G.out[1] = R.dwu;
    G.out_ld = R.dw_ld;
    G.partial = partial;
    G.vec = std::min(row_align(R.dwg, R.dw_ld * sizeof(T)), row_align(R.dwu, R.dw_ld * sizeof(T)));
    CUtensorMap a0, a1;
    GPB_TRY(make_map(dg, 64, BK, &a0));
    GPB_TRY(make_map(du, 64, BK, &a1));
    GPB_TRY((gated_plain<GG_DW, T, D, PL, PD>(a0, a1, x, x, P.tile_n, G, st)));
  }
  const bool bias = R.dbg || R.dbu;
  JoinArgs J{};
  if (P.splits > 1 && (R.dwg || R.dwu))
    J.dw = {partial, P.splits, A.outer, A.inner, R.dw_ld, 2, {R.dwg, R.dwu},
            ceil_div(2 * A.outer * round_up(A.inner, 16), 1024)};
  if (P.splits_x > 1 && R.dx)
    J.dx = {(float*)(ws + P.partial_x), P.splits_x, A.rows, A.inner, R.dx_ld, 1, {R.dx, nullptr},
            ceil_div(A.rows * round_up(A.inner, 16), 1024)};
  J.col_sums = (const float*)(ws + P.sums);
  J.sum_rows = 4 * ceil_div(A.rows, kGgBM);
  J.outer = A.outer;
  J.db[0] = R.dbg;
  J.db[1] = R.dbu;
  const int64_t grid = J.dw.blocks + J.dx.blocks + (bias ? ceil_div(2 * A.outer, 32) : 0);
  if (grid > 0) {
    gated_join_kernel<T><<<(unsigned)grid, 1024, 0, st>>>(J);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

template <typename T, typename D, int PL>
static int gated_backward(const GatedArgs& A, const GatedGrads& R, char* ws, const GatedPlan& P,
                          cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (P.few) {
    const bool vec = gated_vec<T>(A) && (!(R.dwg || R.dwu) || R.dw_ld % V == 0) &&
                     aligned16(R.dwg) && aligned16(R.dwu);
    return vec ? gated_rows_backward<T, V>(A, R, P, ws, st)
               : gated_rows_backward<T, 1>(A, R, P, ws, st);
  }
  if constexpr (PL == 1)
    if (P.planes_d == 2) return gated_backward_tc<T, D, 1, 2>(A, R, ws, P, st);
  return gated_backward_tc<T, D, PL, PL>(A, R, ws, P, st);
}

static int gated_check(int32_t dtype, int64_t rows, int64_t inner, int64_t outer) {
  GPB_REQUIRE(dtype_ok(dtype), GPB_ERR_INVALID, "unknown element type %d", dtype);
  GPB_REQUIRE(rows >= 0 && inner >= 1 && outer >= 1, GPB_ERR_INVALID,
              "gated unit needs rows >= 0, inner >= 1 and outer >= 1, got %lld, %lld, %lld",
              (long long)rows, (long long)inner, (long long)outer);
  GPB_REQUIRE(rows <= ((int64_t)1 << 30) && inner <= (1 << 20) && outer <= (1 << 20),
              GPB_ERR_INVALID, "gated unit sizes %lld, %lld, %lld are too large (2^30, 2^20, 2^20)",
              (long long)rows, (long long)inner, (long long)outer);
  GPB_REQUIRE(rows * std::max(inner, outer) <= ((int64_t)1 << 40), GPB_ERR_INVALID,
              "gated unit of %lld rows is too large", (long long)rows);
  return GPB_OK;
}

}  // namespace gpb

using namespace gpb;

extern "C" {

int gpb_feature_status(int32_t device, int32_t* status_out) {
  clear_error();
  GPB_REQUIRE(status_out, GPB_ERR_INVALID, "null output");
  *status_out = DEV_OK;
  GPB_DEVICE_SCOPE(device);
  int word = 0;
  const int zero = 0;
  GPB_CHECK_CUDA(cudaDeviceSynchronize());
  GPB_CHECK_CUDA(cudaMemcpyFromSymbol(&word, g_feature_err, sizeof(word)));
  if (word != DEV_OK) GPB_CHECK_CUDA(cudaMemcpyToSymbol(g_feature_err, &zero, sizeof(zero)));
  *status_out = word;
  return GPB_OK;
}

int gpb_gated_unit_workspace(int32_t dtype, int64_t rows, int64_t inner, int64_t outer,
                             int32_t backward, int64_t* bytes_out) {
  clear_error();
  GPB_REQUIRE(bytes_out, GPB_ERR_INVALID, "null output");
  GPB_TRY(gated_check(dtype, rows, inner, outer));
  *bytes_out = workspace_need(gated_plan(rows, inner, outer, dtype, backward != 0));
  return GPB_OK;
}

int gpb_gated_unit(int32_t device, void* stream, int32_t dtype, int32_t activation, int64_t rows,
                   int64_t inner, int64_t outer, void* out_dev, int64_t out_ld, const void* x_dev,
                   int64_t x_ld, const void* w_gate_dev, const void* w_up_dev, int64_t w_ld,
                   const void* b_gate_dev, const void* b_up_dev, void* workspace_dev,
                   int64_t workspace_bytes) {
  clear_error();
  GPB_TRY(gated_check(dtype, rows, inner, outer));
  GPB_REQUIRE(activation >= GPB_ACT_SILU && activation <= GPB_ACT_TANH, GPB_ERR_INVALID,
              "unknown activation %d", activation);
  if (rows == 0) return GPB_OK;
  const int es = dtype_bytes(dtype);
  GPB_REQUIRE(out_dev && x_dev && w_gate_dev && w_up_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(x_ld >= inner && w_ld >= inner && out_ld >= outer, GPB_ERR_INVALID,
              "leading dimension below the column count");
  GPB_REQUIRE(elem_aligned(out_dev, es) && elem_aligned(x_dev, es) && elem_aligned(w_gate_dev, es) &&
                  elem_aligned(w_up_dev, es) && elem_aligned(b_gate_dev, es) &&
                  elem_aligned(b_up_dev, es),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const Extent out = block_extent(out_dev, rows, outer, out_ld, es);
  const Extent in[] = {block_extent(x_dev, rows, inner, x_ld, es),
                       block_extent(w_gate_dev, outer, inner, w_ld, es),
                       block_extent(w_up_dev, outer, inner, w_ld, es), flat_extent(b_gate_dev, outer * es),
                       flat_extent(b_up_dev, outer * es)};
  for (const Extent& i : in)
    GPB_REQUIRE(!overlaps(out, i), GPB_ERR_INVALID, "out overlaps an input");
  const GatedPlan P = gated_plan(rows, inner, outer, dtype, false);
  const int64_t need = workspace_need(P);
  GPB_REQUIRE(need == 0 || (workspace_dev && workspace_bytes >= need), GPB_ERR_INVALID,
              "gated unit needs a workspace of %lld bytes, got %lld", (long long)need,
              (long long)(workspace_dev ? workspace_bytes : 0));
  GPB_REQUIRE(aligned16(workspace_dev), GPB_ERR_INVALID, "workspace is not 16-byte aligned");
  const Extent ws_extent = flat_extent(workspace_dev, need);
  bool shared = overlaps(ws_extent, out);
  for (const Extent& i : in) shared = shared || overlaps(ws_extent, i);
  GPB_REQUIRE(!shared, GPB_ERR_INVALID, "the workspace overlaps an input or out");
  GPB_DEVICE_SCOPE(device);
  GatedArgs A{};
  A.x = x_dev;
  A.wg = w_gate_dev;
  A.wu = w_up_dev;
  A.bg = b_gate_dev;
  A.bu = b_up_dev;
  A.out = out_dev;
  A.x_ld = x_ld;
  A.w_ld = w_ld;
  A.out_ld = out_ld;
  A.rows = rows;
  A.inner = inner;
  A.outer = outer;
  A.act = activation;
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = workspace_base(workspace_dev);
  switch (dtype) {
    case GPB_DTYPE_F32:
      return gated_forward<float, __nv_bfloat16, 3>(A, ws, P, st);
    case GPB_DTYPE_F16: return gated_forward<__half, __half, 1>(A, ws, P, st);
    default:
      return gated_forward<__nv_bfloat16, __nv_bfloat16, 1>(A, ws, P, st);
  }
}

int gpb_gated_unit_backward(int32_t device, void* stream, int32_t dtype, int32_t activation,
                            int64_t rows, int64_t inner, int64_t outer, const void* dout_dev,
                            int64_t dout_ld, const void* x_dev, int64_t x_ld,
                            const void* w_gate_dev, const void* w_up_dev, int64_t w_ld,
                            const void* b_gate_dev, const void* b_up_dev, void* dx_dev,
                            int64_t dx_ld, void* dw_gate_dev, void* dw_up_dev, int64_t dw_ld,
                            void* db_gate_dev, void* db_up_dev, void* workspace_dev,
                            int64_t workspace_bytes) {
  clear_error();
  GPB_TRY(gated_check(dtype, rows, inner, outer));
  GPB_REQUIRE(activation >= GPB_ACT_SILU && activation <= GPB_ACT_TANH, GPB_ERR_INVALID,
              "unknown activation %d", activation);
  const int es = dtype_bytes(dtype);
  GPB_REQUIRE((!dx_dev || dx_ld >= inner) && (!(dw_gate_dev || dw_up_dev) || dw_ld >= inner),
              GPB_ERR_INVALID, "leading dimension below the column count");
  GPB_REQUIRE(elem_aligned(dx_dev, es) && elem_aligned(dw_gate_dev, es) &&
                  elem_aligned(dw_up_dev, es) && elem_aligned(db_gate_dev, es) &&
                  elem_aligned(db_up_dev, es),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    GPB_DEVICE_SCOPE(device);
    for (void* w : {dw_gate_dev, dw_up_dev})
      if (w) GPB_CHECK_CUDA(cudaMemset2DAsync(w, dw_ld * es, 0, inner * es, outer, st));
    for (void* b : {db_gate_dev, db_up_dev})
      if (b) GPB_CHECK_CUDA(cudaMemsetAsync(b, 0, outer * es, st));
    return GPB_OK;
  }
  GPB_REQUIRE(dx_dev || dw_gate_dev || dw_up_dev || db_gate_dev || db_up_dev, GPB_ERR_INVALID,
              "no output was asked for");
  GPB_REQUIRE(dout_dev && x_dev && w_gate_dev && w_up_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(x_ld >= inner && w_ld >= inner && dout_ld >= outer, GPB_ERR_INVALID,
              "leading dimension below the column count");
  GPB_REQUIRE(elem_aligned(dout_dev, es) && elem_aligned(x_dev, es) &&
                  elem_aligned(w_gate_dev, es) && elem_aligned(w_up_dev, es) &&
                  elem_aligned(b_gate_dev, es) && elem_aligned(b_up_dev, es),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const GatedPlan P = gated_plan(rows, inner, outer, dtype, true);
  const int64_t need = workspace_need(P);
  GPB_REQUIRE(workspace_dev && workspace_bytes >= need, GPB_ERR_INVALID,
              "the backward pass needs a workspace of %lld bytes, got %lld", (long long)need,
              (long long)(workspace_dev ? workspace_bytes : 0));
  GPB_REQUIRE(aligned16(workspace_dev), GPB_ERR_INVALID, "workspace is not 16-byte aligned");
  {
    // Outputs and the workspace are written while inputs are still read: none may share memory.
    const int64_t bb = outer * es;
    const Extent in[] = {block_extent(dout_dev, rows, outer, dout_ld, es),
                         block_extent(x_dev, rows, inner, x_ld, es),
                         block_extent(w_gate_dev, outer, inner, w_ld, es),
                         block_extent(w_up_dev, outer, inner, w_ld, es), flat_extent(b_gate_dev, bb),
                         flat_extent(b_up_dev, bb)};
    const Extent out[] = {block_extent(dx_dev, rows, inner, dx_ld, es),
                          block_extent(dw_gate_dev, outer, inner, dw_ld, es),
                          block_extent(dw_up_dev, outer, inner, dw_ld, es), flat_extent(db_gate_dev, bb),
                          flat_extent(db_up_dev, bb), flat_extent(workspace_dev, need)};
    for (int o = 0; o < 6; ++o) {
      for (const Extent& i : in)
        GPB_REQUIRE(!overlaps(out[o], i), GPB_ERR_INVALID,
                    "an output or the workspace overlaps an input");
      for (int q = 0; q < o; ++q)
        GPB_REQUIRE(!overlaps(out[o], out[q]), GPB_ERR_INVALID,
                    "two outputs (or an output and the workspace) overlap");
    }
  }
  GPB_DEVICE_SCOPE(device);
  GatedArgs A{};
  A.x = x_dev;
  A.wg = w_gate_dev;
  A.wu = w_up_dev;
  A.bg = b_gate_dev;
  A.bu = b_up_dev;
  A.dout = dout_dev;
  A.x_ld = x_ld;
  A.w_ld = w_ld;
  A.dout_ld = dout_ld;
  A.rows = rows;
  A.inner = inner;
  A.outer = outer;
  A.act = activation;
  GatedGrads G{dx_dev, dx_ld, dw_gate_dev, dw_up_dev, dw_ld, db_gate_dev, db_up_dev};
  char* ws = workspace_base(workspace_dev);
  switch (dtype) {
    case GPB_DTYPE_F32:
      return gated_backward<float, __nv_bfloat16, 3>(A, G, ws, P, st);
    case GPB_DTYPE_F16: return gated_backward<__half, __half, 1>(A, G, ws, P, st);
    default:
      return gated_backward<__nv_bfloat16, __nv_bfloat16, 1>(A, G, ws, P, st);
  }
}

}  // extern "C"
