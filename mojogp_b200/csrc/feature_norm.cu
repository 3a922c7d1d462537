// Layer norm over the columns of a row-major [rows][cols] block, forward and backward.
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w,  xhat = (x - mean) rstd,  dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum_rows dy xhat,  db = sum_rows dy
// Everything is held in fp32 and rounded once, to the output's type. The variance is the second
// pass over the row's registers (no E[x^2] - mean^2 cancellation). dw and db are summed in a fixed
// order (per block in row order, then over blocks), so results repeat bit for bit.
//
// A row belongs to TPR threads (a power of two: part of a warp, or the block), each of which keeps
// R vectors of VEC elements in registers: x and dy are read once and dx is written once.
#include <algorithm>

#include "features.cuh"

namespace gpb {

struct NormArgs {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* out;  // y or dx
  float* mean;
  float* rstd;
  float* partial;  // [blocks][2][cols] dw, db sums
  int64_t x_ld, dy_ld, out_ld;
  int64_t rows;
  int32_t cols;
  int32_t tpr;
  float eps;
};

// Sums (a, b) over the TPR threads of a row; every thread of the block takes part. `flip` alternates
// the shared buffer so that one barrier per call is enough.
__device__ __forceinline__ void row_sum2(float& a, float& b, int tpr, int flip) {
  const int width = tpr < 32 ? tpr : 32;
  for (int o = width >> 1; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (tpr > 32) {
    __shared__ float2 part[2][32];
    const int warp = threadIdx.x >> 5, warps = tpr >> 5;
    const int first = warp & ~(warps - 1);  // first warp of this row
    if ((threadIdx.x & 31) == 0) part[flip][warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) {
      const float2 p = part[flip][first + w];
      a += p.x;
      b += p.y;
    }
  }
}

template <typename T, typename W, int VEC, int R>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs A) {
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < A.rows;
  const T* x = (const T*)A.x + (live ? row : 0) * A.x_ld;
  float v[R][VEC];
  float s = 0.f, unused = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * tpr + lane) * VEC;
    if (live && c < A.cols) {
      load_vec<T, VEC>(x + c, v[r]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[r][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s += v[r][i];
  }
  row_sum2(s, unused, tpr, 0);
  const float mean = s / (float)A.cols;
  float q = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = (r * tpr + lane) * VEC < A.cols;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[r][i] -= mean;
      q = in ? fmaf(v[r][i], v[r][i], q) : q;
    }
  }
  row_sum2(q, unused, tpr, 1);
  const float rstd = 1.f / sqrtf(q / (float)A.cols + A.eps);
  if (!live) return;
  if (lane == 0) {
    if (A.mean) A.mean[row] = mean;
    if (A.rstd) A.rstd[row] = rstd;
  }
  T* y = (T*)A.out + row * A.out_ld;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * tpr + lane) * VEC;
    if (c >= A.cols) break;
    float w[VEC], b[VEC], o[VEC];
    if (A.w) load_vec<W, VEC>((const W*)A.w + c, w);
    if (A.b) load_vec<W, VEC>((const W*)A.b + c, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      o[i] = v[r][i] * rstd;
      if (A.w) o[i] *= w[i];
      if (A.b) o[i] += b[i];
    }
    store_vec<T, VEC>(y + c, o);
  }
}

// Rows too wide for registers: one block per row, x read three times (the second and third from L2).
template <typename T, typename W>
__global__ void __launch_bounds__(1024) norm_forward_wide_kernel(const NormArgs A) {
  const int64_t row = blockIdx.x;
  const T* x = (const T*)A.x + row * A.x_ld;
  float s = 0.f, unused = 0.f;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) s += to_f(x[c]);
  row_sum2(s, unused, blockDim.x, 0);
  const float mean = s / (float)A.cols;
  float q = 0.f;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    const float d = to_f(x[c]) - mean;
    q = fmaf(d, d, q);
  }
  row_sum2(q, unused, blockDim.x, 1);
  const float rstd = 1.f / sqrtf(q / (float)A.cols + A.eps);
  if (threadIdx.x == 0) {
    if (A.mean) A.mean[row] = mean;
    if (A.rstd) A.rstd[row] = rstd;
  }
  T* y = (T*)A.out + row * A.out_ld;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    float o = (to_f(x[c]) - mean) * rstd;
    if (A.w) o *= to_f(((const W*)A.w)[c]);
    if (A.b) o += to_f(((const W*)A.b)[c]);
    y[c] = from_f<T>(o);
  }
}

// Backward with the weight gradients: a fixed number of blocks walks the rows, each thread adding
// the dw and db of its columns; the block's sums go to A.partial.
template <typename T, typename W, int VEC, int R, bool PARAMS>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormArgs A) {
  extern __shared__ float row_sums[];  // [slots][2][cols] when the block holds several rows
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr;
  float dw[R][VEC], db[R][VEC];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[r][i] = db[r][i] = 0.f;
  int flip = 0;
  const float inv = 1.f / (float)A.cols;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows;
       base += (int64_t)gridDim.x * groups) {
    const int64_t row = base + threadIdx.x / tpr;
    const bool live = row < A.rows;
    const int64_t rr = live ? row : 0;
    const T* x = (const T*)A.x + rr * A.x_ld;
    const T* dy = (const T*)A.dy + rr * A.dy_ld;
    const float mean = A.mean[rr], rstd = A.rstd[rr];
    float xh[R][VEC], g[R][VEC];
    float sg = 0.f, sgx = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = (r * tpr + lane) * VEC;
      if (live && c < A.cols) {
        load_vec<T, VEC>(x + c, xh[r]);
        load_vec<T, VEC>(dy + c, g[r]);
        float w[VEC];
        if (A.w) load_vec<W, VEC>((const W*)A.w + c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          xh[r][i] = (xh[r][i] - mean) * rstd;
          if constexpr (PARAMS) {
            dw[r][i] = fmaf(g[r][i], xh[r][i], dw[r][i]);
            db[r][i] += g[r][i];
          }
          if (A.w) g[r][i] *= w[i];
          sg += g[r][i];
          sgx = fmaf(g[r][i], xh[r][i], sgx);
        }
      }
    }
    if (A.out) {
      row_sum2(sg, sgx, tpr, flip);
      flip ^= 1;
      const float mg = sg * inv, mgx = sgx * inv;
      if (live) {
        T* dx = (T*)A.out + row * A.out_ld;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int c = (r * tpr + lane) * VEC;
          if (c < A.cols) {
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = rstd * (g[r][i] - mg - xh[r][i] * mgx);
            store_vec<T, VEC>(dx + c, o);
          }
        }
      }
    }
  }
  if constexpr (PARAMS) {
    float* part = A.partial + (int64_t)blockIdx.x * 2 * A.cols;
    if (groups == 1) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int c = (r * tpr + lane) * VEC;
        if (c < A.cols) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            part[c + i] = dw[r][i];
            part[A.cols + c + i] = db[r][i];
          }
        }
      }
      return;
    }
    // Several rows at a time: add the rows of each warp, then over the slots (a warp, or the warps
    // of one row).
    const int slots = tpr < 32 ? blockDim.x >> 5 : groups;
    float* mine = row_sums + (int64_t)(threadIdx.x / (tpr < 32 ? 32 : tpr)) * 2 * A.cols;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = (r * tpr + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        for (int o = tpr; o < 32; o <<= 1) {
          dw[r][i] += __shfl_xor_sync(0xffffffffu, dw[r][i], o);
          db[r][i] += __shfl_xor_sync(0xffffffffu, db[r][i], o);
        }
        if ((threadIdx.x & 31) < tpr && c < A.cols) {  // always true for whole warps
          mine[c + i] = dw[r][i];
          mine[A.cols + c + i] = db[r][i];
        }
      }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < 2 * A.cols; q += blockDim.x) {
      float s = 0.f;
      for (int w = 0; w < slots; ++w) s += row_sums[(int64_t)w * 2 * A.cols + q];
      part[q] = s;
    }
  }
}

// dx of rows too wide for registers: x and dy are read twice.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(const NormArgs A) {
  const int64_t row = blockIdx.x;
  const T* x = (const T*)A.x + row * A.x_ld;
  const T* dy = (const T*)A.dy + row * A.dy_ld;
  const float mean = A.mean[row], rstd = A.rstd[row];
  float sg = 0.f, sgx = 0.f;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    float g = to_f(dy[c]);
    if (A.w) g *= to_f(((const W*)A.w)[c]);
    sg += g;
    sgx = fmaf(g, (to_f(x[c]) - mean) * rstd, sgx);
  }
  row_sum2(sg, sgx, blockDim.x, 0);
  const float mg = sg / (float)A.cols, mgx = sgx / (float)A.cols;
  T* dx = (T*)A.out + row * A.out_ld;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    float g = to_f(dy[c]);
    if (A.w) g *= to_f(((const W*)A.w)[c]);
    dx[c] = from_f<T>(rstd * (g - mg - (to_f(x[c]) - mean) * rstd * mgx));
  }
}

// dw and db partial sums of wide rows, column by column: blockIdx.x = 256 columns, blockIdx.y = a
// range of rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_params_wide_kernel(const NormArgs A) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= A.cols) return;
  const int64_t per = (A.rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per;
  const int64_t r1 = r0 + per < A.rows ? r0 + per : A.rows;
  float dw = 0.f, db = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_f(((const T*)A.dy)[r * A.dy_ld + c]);
    const float xh = (to_f(((const T*)A.x)[r * A.x_ld + c]) - A.mean[r]) * A.rstd[r];
    dw = fmaf(g, xh, dw);
    db += g;
  }
  float* part = A.partial + (int64_t)blockIdx.y * 2 * A.cols;
  part[c] = dw;
  part[A.cols + c] = db;
}

// dw and db from the blocks' partial sums: 32 columns per block, 8 threads along the blocks of each.
template <typename W>
__global__ void __launch_bounds__(256) norm_params_sum_kernel(const float* __restrict__ partial,
                                                              int blocks, int cols, W* dw, W* db) {
  __shared__ float sums[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float s = 0.f;
  if (c < 2 * cols)
    for (int b = part; b < blocks; b += 8) s += partial[(int64_t)b * 2 * cols + c];
  sums[part][threadIdx.x & 31] = s;
  __syncthreads();
  if (part == 0 && c < 2 * cols) {
    for (int q = 1; q < 8; ++q) s += sums[q][threadIdx.x & 31];
    W* dst = c < cols ? dw : db;
    if (dst) dst[c < cols ? c : c - cols] = from_f<W>(s);
  }
}

// ------------------------------------------------------------------ host
// Threads per row and vectors per thread for `nvec` vectors: the widest part of a warp first, then
// blocks of warps, growing R only once the row has `max_tpr` threads. Returns R, or 0 when the row
// does not fit max_tpr threads with max_r vectors each.
static int norm_shape(int64_t nvec, int max_tpr, int max_r, int* tpr) {
  int t = 1;
  while (t < max_tpr && t < nvec) t <<= 1;
  int r = 1;
  while ((int64_t)t * r < nvec) r <<= 1;
  *tpr = t;
  return r <= max_r ? r : 0;
}

// Blocks of the backward pass (each writes one partial row of 2 cols sums), a function of the sizes
// alone so that the workspace query and the launch agree.
static int norm_blocks(int64_t rows, int64_t cols) {
  int64_t b = kFeatSMs * (cols <= 1024 ? 8 : cols <= 4096 ? 4 : 2);
  return (int)(b < rows ? b : (rows > 0 ? rows : 1));
}

template <typename T, typename W, int VEC>
static int norm_forward_launch(NormArgs A, cudaStream_t st) {
  constexpr int kMaxR = VEC == 1 ? 8 : 32 / VEC;
  int tpr = 1;
  const int r = norm_shape(ceil_div(A.cols, VEC), 1024, kMaxR, &tpr);
  A.tpr = tpr;
  if (r == 0) {
    norm_forward_wide_kernel<T, W><<<(unsigned)A.rows, 1024, 0, st>>>(A);
  } else {
    const int threads = tpr > 128 ? tpr : 128;
    const unsigned grid = (unsigned)ceil_div(A.rows, threads / tpr);
    switch (r) {
      case 1: norm_forward_kernel<T, W, VEC, 1><<<grid, threads, 0, st>>>(A); break;
      case 2: norm_forward_kernel<T, W, VEC, 2><<<grid, threads, 0, st>>>(A); break;
      case 4: norm_forward_kernel<T, W, VEC, 4><<<grid, threads, 0, st>>>(A); break;
      default: norm_forward_kernel<T, W, VEC, kMaxR><<<grid, threads, 0, st>>>(A);
    }
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, typename W, int VEC, bool PARAMS>
static int norm_backward_vec(NormArgs A, int* blocks, cudaStream_t st, bool* done) {
  constexpr int kMaxR = VEC == 1 ? 8 : 16 / VEC;
  int tpr = 1;
  const int r = norm_shape(ceil_div(A.cols, VEC), 512, kMaxR, &tpr);
  *done = r != 0;
  if (r == 0) return GPB_OK;
  A.tpr = tpr;
  const int threads = tpr > 256 ? tpr : 256;
  // At most 16 KB: a row of fewer threads than the block has one vector per thread.
  const int slots = tpr < 32 ? threads / 32 : threads / tpr;
  const size_t smem = PARAMS && tpr < threads ? (size_t)slots * 2 * A.cols * sizeof(float) : 0;
  const int grid = (int)std::min<int64_t>(*blocks, ceil_div(A.rows, threads / tpr));
  *blocks = grid;
  switch (r) {
    case 1: norm_backward_kernel<T, W, VEC, 1, PARAMS><<<grid, threads, smem, st>>>(A); break;
    case 2: norm_backward_kernel<T, W, VEC, 2, PARAMS><<<grid, threads, smem, st>>>(A); break;
    case 4: norm_backward_kernel<T, W, VEC, 4 <= kMaxR ? 4 : kMaxR, PARAMS><<<grid, threads, smem, st>>>(A); break;
    default: norm_backward_kernel<T, W, VEC, kMaxR, PARAMS><<<grid, threads, smem, st>>>(A);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, typename W, int VEC>
static int norm_backward_launch(NormArgs A, W* dw, W* db, cudaStream_t st) {
  const bool params = dw || db;
  int blocks = norm_blocks(A.rows, A.cols);
  bool done = false;
  if (params)
    GPB_TRY((norm_backward_vec<T, W, VEC, true>(A, &blocks, st, &done)));
  else
    GPB_TRY((norm_backward_vec<T, W, VEC, false>(A, &blocks, st, &done)));
  if (!done) {
    // The parameter sums read x and dy before dx may overwrite them in place.
    if (params) {
      blocks = std::min(blocks, 64);
      norm_params_wide_kernel<T>
          <<<dim3((unsigned)ceil_div(A.cols, 256), blocks), 256, 0, st>>>(A);
      GPB_CHECK_CUDA(cudaGetLastError());
    }
    if (A.out) {
      norm_backward_wide_kernel<T, W><<<(unsigned)A.rows, 1024, 0, st>>>(A);
      GPB_CHECK_CUDA(cudaGetLastError());
    }
  }
  if (params) {
    norm_params_sum_kernel<W><<<(unsigned)ceil_div(2 * (int64_t)A.cols, 32), 256, 0, st>>>(
        A.partial, blocks, A.cols, dw, db);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

template <typename T, typename W>
static int norm_forward_typed(const NormArgs& A, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = A.cols % VEC == 0 && A.x_ld % VEC == 0 && A.out_ld % VEC == 0 &&
                   aligned16(A.x) && aligned16(A.out) && aligned16(A.w) && aligned16(A.b);
  return vec ? norm_forward_launch<T, W, VEC>(A, st) : norm_forward_launch<T, W, 1>(A, st);
}

template <typename T, typename W>
static int norm_backward_typed(const NormArgs& A, void* dw, void* db, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = A.cols % VEC == 0 && A.x_ld % VEC == 0 && A.dy_ld % VEC == 0 &&
                   (!A.out || A.out_ld % VEC == 0) && aligned16(A.x) && aligned16(A.dy) &&
                   aligned16(A.out) && aligned16(A.w);
  return vec ? norm_backward_launch<T, W, VEC>(A, (W*)dw, (W*)db, st)
             : norm_backward_launch<T, W, 1>(A, (W*)dw, (W*)db, st);
}

static int norm_check(int32_t dtype, int32_t param_dtype, int64_t rows, int64_t cols) {
  GPB_REQUIRE(dtype_ok(dtype), GPB_ERR_INVALID, "unknown element type %d", dtype);
  GPB_REQUIRE(param_dtype == dtype || param_dtype == GPB_DTYPE_F32, GPB_ERR_INVALID,
              "weight and bias must be float32 or of x's type");
  GPB_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), GPB_ERR_INVALID, "bad row count %lld",
              (long long)rows);
  GPB_REQUIRE(cols >= 1 && cols <= (1 << 24), GPB_ERR_INVALID,
              "layer norm needs 1 to 16777216 columns, got %lld", (long long)cols);
  return GPB_OK;
}

}  // namespace gpb

using namespace gpb;

extern "C" {

int gpb_layer_norm(int32_t device, void* stream, int32_t dtype, int32_t param_dtype, int64_t rows,
                   int64_t cols, void* out_dev, int64_t out_ld, const void* x_dev, int64_t x_ld,
                   const void* weight_dev, const void* bias_dev, float eps, float* mean_dev,
                   float* rstd_dev) {
  clear_error();
  GPB_TRY(norm_check(dtype, param_dtype, rows, cols));
  GPB_REQUIRE(eps >= 0.f && eps < 3.0e38f, GPB_ERR_INVALID, "eps must be finite and >= 0");
  if (rows == 0) return GPB_OK;
  const int es = dtype_bytes(dtype), ps = dtype_bytes(param_dtype);
  GPB_REQUIRE(out_dev && x_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(out_ld >= cols && x_ld >= cols, GPB_ERR_INVALID,
              "leading dimension below the %lld columns", (long long)cols);
  GPB_REQUIRE(elem_aligned(out_dev, es) && elem_aligned(x_dev, es) &&
                  elem_aligned(weight_dev, ps) && elem_aligned(bias_dev, ps) &&
                  elem_aligned(mean_dev, 4) && elem_aligned(rstd_dev, 4),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  GPB_REQUIRE((out_dev == x_dev && out_ld == x_ld) ||
                  !overlaps(out_dev, span_bytes(rows, cols, out_ld, es), x_dev,
                            span_bytes(rows, cols, x_ld, es)),
              GPB_ERR_INVALID, "out overlaps x (in place needs the same pointer and stride)");
  GPB_DEVICE_SCOPE(device);
  NormArgs A{};
  A.x = x_dev;
  A.w = weight_dev;
  A.b = bias_dev;
  A.out = out_dev;
  A.mean = mean_dev;
  A.rstd = rstd_dev;
  A.x_ld = x_ld;
  A.out_ld = out_ld;
  A.rows = rows;
  A.cols = (int32_t)cols;
  A.eps = eps;
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = param_dtype == GPB_DTYPE_F32;
  switch (dtype) {
    case GPB_DTYPE_F32: return norm_forward_typed<float, float>(A, st);
    case GPB_DTYPE_F16:
      return wide ? norm_forward_typed<__half, float>(A, st)
                  : norm_forward_typed<__half, __half>(A, st);
    default:
      return wide ? norm_forward_typed<__nv_bfloat16, float>(A, st)
                  : norm_forward_typed<__nv_bfloat16, __nv_bfloat16>(A, st);
  }
}

int gpb_layer_norm_workspace(int64_t rows, int64_t cols, int64_t* bytes_out) {
  clear_error();
  GPB_REQUIRE(bytes_out, GPB_ERR_INVALID, "null output");
  GPB_TRY(norm_check(GPB_DTYPE_F32, GPB_DTYPE_F32, rows, cols));
  *bytes_out = (int64_t)norm_blocks(rows, cols) * 2 * cols * (int64_t)sizeof(float);
  return GPB_OK;
}

int gpb_layer_norm_backward(int32_t device, void* stream, int32_t dtype, int32_t param_dtype,
                            int64_t rows, int64_t cols, void* dx_dev, int64_t dx_ld,
                            const void* dout_dev, int64_t dout_ld, const void* x_dev, int64_t x_ld,
                            const float* mean_dev, const float* rstd_dev, const void* weight_dev,
                            void* dweight_dev, void* dbias_dev, void* workspace_dev,
                            int64_t workspace_bytes) {
  clear_error();
  GPB_TRY(norm_check(dtype, param_dtype, rows, cols));
  const bool params = dweight_dev || dbias_dev;
  const int es = dtype_bytes(dtype), ps = dtype_bytes(param_dtype);
  GPB_REQUIRE(dx_dev || params, GPB_ERR_INVALID, "no output was asked for");
  GPB_REQUIRE(elem_aligned(dweight_dev, ps) && elem_aligned(dbias_dev, ps), GPB_ERR_INVALID,
              "pointer is not aligned to its element type");
  if (rows == 0) {
    GPB_DEVICE_SCOPE(device);
    if (dweight_dev) GPB_CHECK_CUDA(cudaMemsetAsync(dweight_dev, 0, cols * ps, (cudaStream_t)stream));
    if (dbias_dev) GPB_CHECK_CUDA(cudaMemsetAsync(dbias_dev, 0, cols * ps, (cudaStream_t)stream));
    return GPB_OK;
  }
  GPB_REQUIRE(dout_dev && x_dev && mean_dev && rstd_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(dout_ld >= cols && x_ld >= cols && (!dx_dev || dx_ld >= cols), GPB_ERR_INVALID,
              "leading dimension below the %lld columns", (long long)cols);
  GPB_REQUIRE(elem_aligned(dx_dev, es) && elem_aligned(dout_dev, es) && elem_aligned(x_dev, es) &&
                  elem_aligned(weight_dev, ps) && elem_aligned(mean_dev, 4) &&
                  elem_aligned(rstd_dev, 4),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const int64_t dxb = dx_dev ? span_bytes(rows, cols, dx_ld, es) : 0;
  GPB_REQUIRE((dx_dev == dout_dev && dx_ld == dout_ld) ||
                  !overlaps(dx_dev, dxb, dout_dev, span_bytes(rows, cols, dout_ld, es)),
              GPB_ERR_INVALID, "dx overlaps dout (in place needs the same pointer and stride)");
  GPB_REQUIRE((dx_dev == x_dev && dx_ld == x_ld) ||
                  !overlaps(dx_dev, dxb, x_dev, span_bytes(rows, cols, x_ld, es)),
              GPB_ERR_INVALID, "dx overlaps x (in place needs the same pointer and stride)");
  if (params) {
    const int64_t need = (int64_t)norm_blocks(rows, cols) * 2 * cols * (int64_t)sizeof(float);
    GPB_REQUIRE(workspace_dev && workspace_bytes >= need, GPB_ERR_INVALID,
                "the weight gradients need a workspace of %lld bytes, got %lld", (long long)need,
                (long long)(workspace_dev ? workspace_bytes : 0));
    GPB_REQUIRE(aligned16(workspace_dev), GPB_ERR_INVALID, "workspace is not 16-byte aligned");
  }
  GPB_DEVICE_SCOPE(device);
  NormArgs A{};
  A.x = x_dev;
  A.dy = dout_dev;
  A.w = weight_dev;
  A.out = dx_dev;
  A.mean = const_cast<float*>(mean_dev);
  A.rstd = const_cast<float*>(rstd_dev);
  A.partial = (float*)workspace_dev;
  A.x_ld = x_ld;
  A.dy_ld = dout_ld;
  A.out_ld = dx_ld;
  A.rows = rows;
  A.cols = (int32_t)cols;
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = param_dtype == GPB_DTYPE_F32;
  switch (dtype) {
    case GPB_DTYPE_F32: return norm_backward_typed<float, float>(A, dweight_dev, dbias_dev, st);
    case GPB_DTYPE_F16:
      return wide ? norm_backward_typed<__half, float>(A, dweight_dev, dbias_dev, st)
                  : norm_backward_typed<__half, __half>(A, dweight_dev, dbias_dev, st);
    default:
      return wide
                 ? norm_backward_typed<__nv_bfloat16, float>(A, dweight_dev, dbias_dev, st)
                 : norm_backward_typed<__nv_bfloat16, __nv_bfloat16>(A, dweight_dev, dbias_dev, st);
  }
}

}  // extern "C"
