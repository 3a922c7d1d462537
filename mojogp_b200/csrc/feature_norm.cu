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

// Sums each of N values over the TPR threads of a row; every thread of the block takes part. `flip`
// alternates the shared buffer so that one barrier per call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, int flip) {
  const int width = tpr < 32 ? tpr : 32;
  for (int o = width >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
  if (tpr > 32) {
    __shared__ float part[2][N][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = tpr >> 5;
    const int first = warp & ~(warps - 1);  // first warp of this row
    if (lane == 0)
#pragma unroll
      for (int q = 0; q < N; ++q) part[flip][q][warp] = v[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = part[flip][q][first + (lane & (warps - 1))];
    for (int o = warps >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int q = 0; q < N; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
  }
}

// 1 / sqrt(v), v >= 0: the hardware's estimate and one Newton step (about 1 ulp; a division and a
// square root cost 30 instructions a row).
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  return v > 0.f ? fmaf(fmaf(-0.5f * v * r, r, 0.5f), r, r) : r;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows of at most 32 vectors: TPR threads (part of a warp) hold one vector each of RPT rows, so that
// RPT loads are in flight where one row's would leave HBM idle.
template <typename T, typename W, int VEC, int RPT>
__global__ void __launch_bounds__(128) norm_forward_rows_kernel(const NormArgs A) {
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int group = threadIdx.x / tpr, groups = 128 / tpr;
  const int64_t row0 = (int64_t)blockIdx.x * (groups * RPT) + group;
  const int c = lane * VEC;
  const bool in = c < A.cols;
  float v[RPT][VEC], w[VEC], b[VEC];
#pragma unroll
  for (int u = 0; u < RPT; ++u) {
    const int64_t row = row0 + u * groups;
    if (in && row < A.rows) {
      load_vec<T, VEC>((const T*)A.x + row * A.x_ld + c, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
    }
  }
  if (in && A.w) load_vec<W, VEC>((const W*)A.w + c, w);
  if (in && A.b) load_vec<W, VEC>((const W*)A.b + c, b);
  const float inv = 1.f / (float)A.cols;
  float s[RPT], q[RPT];
#pragma unroll
  for (int u = 0; u < RPT; ++u) {
    s[u] = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[u] += v[u][i];
  }
  row_sum(s, tpr, 0);
#pragma unroll
  for (int u = 0; u < RPT; ++u) {
    s[u] *= inv;
    q[u] = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[u][i] -= s[u];
      q[u] = in ? fmaf(v[u][i], v[u][i], q[u]) : 0.f;
    }
  }
  row_sum(q, tpr, 0);
#pragma unroll
  for (int u = 0; u < RPT; ++u) {
    const int64_t row = row0 + u * groups;
    if (row >= A.rows) break;
    const float rstd = inv_sqrt(fmaf(q[u], inv, A.eps));
    if (lane == 0) {
      if (A.mean) A.mean[row] = s[u];
      if (A.rstd) A.rstd[row] = rstd;
    }
    if (in) {
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        o[i] = v[u][i] * rstd;
        if (A.w) o[i] *= w[i];
        if (A.b) o[i] += b[i];
      }
      store_vec<T, VEC>((T*)A.out + row * A.out_ld + c, o);
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
  float s[1] = {0.f}, q[1] = {0.f};
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
    for (int i = 0; i < VEC; ++i) s[0] += v[r][i];
  }
  row_sum(s, tpr, 0);
  const float mean = s[0] / (float)A.cols;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = (r * tpr + lane) * VEC < A.cols;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[r][i] -= mean;
      q[0] = in ? fmaf(v[r][i], v[r][i], q[0]) : q[0];
    }
  }
  row_sum(q, tpr, 1);
  const float rstd = inv_sqrt(q[0] / (float)A.cols + A.eps);
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
  float s[1] = {0.f}, q[1] = {0.f};
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) s[0] += to_f(x[c]);
  row_sum(s, blockDim.x, 0);
  const float mean = s[0] / (float)A.cols;
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    const float d = to_f(x[c]) - mean;
    q[0] = fmaf(d, d, q[0]);
  }
  row_sum(q, blockDim.x, 1);
  const float rstd = inv_sqrt(q[0] / (float)A.cols + A.eps);
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

// A block's dw and db sums, from every thread's own columns.
template <int VEC, int R>
__device__ __forceinline__ void norm_store_partial(const NormArgs& A, float* row_sums,
                                                   float (&dw)[R][VEC], float (&db)[R][VEC]) {
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr;
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
  // Several rows at a time: add the rows of each warp, then over the slots (a warp, or the warps of
  // one row).
  const int slots = tpr < 32 ? blockDim.x >> 5 : groups;
  float* mine = row_sums + (int64_t)(threadIdx.x / (tpr < 32 ? 32 : tpr)) * 2 * A.cols;
  __syncthreads();  // the memory may have been a ring
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

// Backward with the weight gradients: a fixed number of blocks walks the rows, each thread adding
// the dw and db of its columns; the block's sums go to A.partial. Vector rows: 16-byte cp.async
// copies fill a ring that only their own thread reads (no barrier), and the arithmetic is on fp32
// pairs (FFMA2). Measured at 16384 x 4096 bf16 (403 MB): one column vector per thread on scalar FMAs
// 125 us, issue-bound at 48 instructions an element; two vectors on pairs, which spread a row's
// address, reduction and barrier work over twice the columns, 80 us (5.0 TB/s). What is left is the
// chain of a row's reduction at two blocks per SM (121 registers); a deeper ring changes nothing.
// Rows in flight per thread: what two resident blocks' rings have room for.
template <int R>
constexpr int kNormAhead = R >= 4 ? 2 : 4;

template <typename T, typename W, int VEC, int R, bool PARAMS>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormArgs A) {
  constexpr int SLOTS = kNormAhead<R> + 1;
  constexpr int P = VEC / 2;
  extern __shared__ __align__(16) float row_sums[];  // the ring, then [slots][2][cols]
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr;
  const int64_t step = (int64_t)gridDim.x * groups;
  const int64_t base = (int64_t)blockIdx.x * groups;
  const int64_t first = base + threadIdx.x / tpr;
  const int loops = (int)((A.rows - base + step - 1) / step);  // of the block
  const int mine = first < A.rows ? (int)((A.rows - first + step - 1) / step) : 0;
  const int c0 = lane * VEC, dc = tpr * VEC;
  const T* xf = (const T*)A.x + first * A.x_ld + c0;  // next row to fetch
  const T* df = (const T*)A.dy + first * A.dy_ld + c0;
  T* out = (T*)A.out + first * A.out_ld + c0;
  const float* mp = A.mean + first;
  const float* rp = A.rstd + first;
  const int64_t x_step = step * A.x_ld, dy_step = step * A.dy_ld, out_step = step * A.out_ld;
  const uint32_t stride = blockDim.x * 16, span = R * 2 * stride;
  const uint32_t ring = smem_addr(row_sums) + threadIdx.x * 16;
  const char* ring_p = reinterpret_cast<const char*>(row_sums) + threadIdx.x * 16;
  bool in[R];
#pragma unroll
  for (int r = 0; r < R; ++r) in[r] = c0 + r * dc < A.cols;
  int fetched = 0;
  uint32_t fill = 0;  // byte offset of the slot to fill
  auto fetch = [&]() {
    if (fetched < mine) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (in[r]) {
          copy16(ring + fill + (2 * r) * stride, xf + r * dc);
          copy16(ring + fill + (2 * r + 1) * stride, df + r * dc);
        }
      xf += x_step;
      df += dy_step;
    }
    copy_commit();
    ++fetched;
    fill = fill + span == SLOTS * span ? 0 : fill + span;
  };
  float2 w[R][P], dw[R][P], db[R][P];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = 1.f;
    if (A.w && in[r]) load_vec<W, VEC>((const W*)A.w + c0 + r * dc, t);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      w[r][i] = make_float2(t[2 * i], t[2 * i + 1]);
      dw[r][i] = db[r][i] = make_float2(0.f, 0.f);
    }
  }
#pragma unroll
  for (int s = 0; s < kNormAhead<R>; ++s) fetch();
  const float inv = 1.f / (float)A.cols;
  uint32_t at = 0;
  float mean = 0 < mine ? *mp : 0.f, rstd = 0 < mine ? *rp : 0.f;
  for (int k = 0; k < loops; ++k) {
    copy_wait<kNormAhead<R> - 1>();
    fetch();  // into the slot of the row before this one, whose values are long used
    const float scale = rstd, shift = -mean * rstd;
    if (k + 1 < mine) {
      mp += step;
      rp += step;
      mean = *mp;
      rstd = *rp;
    }
    const bool live = k < mine;
    float2 xh[R][P], g[R][P];
    float2 sg = make_float2(0.f, 0.f), sgx = make_float2(0.f, 0.f);
    const float2 scale2 = make_float2(scale, scale), shift2 = make_float2(shift, shift);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint4 xr = make_uint4(0, 0, 0, 0), dr = make_uint4(0, 0, 0, 0);
      if (live && in[r]) {
        xr = *reinterpret_cast<const uint4*>(ring_p + at + (2 * r) * stride);
        dr = *reinterpret_cast<const uint4*>(ring_p + at + (2 * r + 1) * stride);
      }
      unpack16(xr, xh[r], (const T*)nullptr);
      unpack16(dr, g[r], (const T*)nullptr);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        xh[r][i] = __ffma2_rn(xh[r][i], scale2, shift2);
        if constexpr (PARAMS) {
          dw[r][i] = __ffma2_rn(g[r][i], xh[r][i], dw[r][i]);
          db[r][i] = __fadd2_rn(g[r][i], db[r][i]);
        }
        g[r][i] = __fmul2_rn(g[r][i], w[r][i]);
        sg = __fadd2_rn(g[r][i], sg);
        sgx = __ffma2_rn(g[r][i], xh[r][i], sgx);
      }
    }
    if (A.out) {
      float sums[2] = {sg.x + sg.y, sgx.x + sgx.y};
      row_sum(sums, tpr, k & 1);
      const float mg = -scale * (sums[0] * inv), mgx = -scale * (sums[1] * inv);
      if (live) {
        const float2 mg2 = make_float2(mg, mg), mgx2 = make_float2(mgx, mgx);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float2 o[P];
#pragma unroll
          for (int i = 0; i < P; ++i)
            o[i] = __ffma2_rn(xh[r][i], mgx2, __ffma2_rn(g[r][i], scale2, mg2));
          if (in[r]) *reinterpret_cast<uint4*>(out + r * dc) = pack16(o, (const T*)nullptr);
        }
      }
      out += out_step;
    }
    at = at + span == SLOTS * span ? 0 : at + span;
  }
  copy_wait<0>();
  if constexpr (PARAMS) {
    float a[R][VEC], b[R][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        a[r][2 * i] = dw[r][i].x;
        a[r][2 * i + 1] = dw[r][i].y;
        b[r][2 * i] = db[r][i].x;
        b[r][2 * i + 1] = db[r][i].y;
      }
    norm_store_partial<VEC, R>(A, row_sums, a, b);
  }
}

// The same for rows that are not 16-byte aligned: one element at a time.
template <typename T, typename W, int R, bool PARAMS>
__global__ void __launch_bounds__(512) norm_backward_scalar_kernel(const NormArgs A) {
  extern __shared__ __align__(16) float row_sums[];  // [slots][2][cols]
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr;
  float dw[R][1], db[R][1];
#pragma unroll
  for (int r = 0; r < R; ++r) dw[r][0] = db[r][0] = 0.f;
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
    float xh[R], g[R], sums[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = r * tpr + lane;
      const bool in = live && c < A.cols;
      xh[r] = in ? to_f(x[c]) : 0.f;
      g[r] = in ? to_f(dy[c]) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = r * tpr + lane;
      xh[r] = (xh[r] - mean) * rstd;
      if constexpr (PARAMS) {
        dw[r][0] = fmaf(g[r], xh[r], dw[r][0]);
        db[r][0] += g[r];
      }
      if (A.w && c < A.cols) g[r] *= to_f(((const W*)A.w)[c]);
      sums[0] += g[r];
      sums[1] = fmaf(g[r], xh[r], sums[1]);
    }
    if (A.out) {
      row_sum(sums, tpr, flip);
      flip ^= 1;
      const float mg = sums[0] * inv, mgx = sums[1] * inv;
      if (live) {
        T* dx = (T*)A.out + row * A.out_ld;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int c = r * tpr + lane;
          if (c < A.cols) dx[c] = from_f<T>(rstd * (g[r] - mg - xh[r] * mgx));
        }
      }
    }
  }
  if constexpr (PARAMS) norm_store_partial<1, R>(A, row_sums, dw, db);
}

// dx of rows too wide for registers: x and dy are read twice.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(const NormArgs A) {
  const int64_t row = blockIdx.x;
  const T* x = (const T*)A.x + row * A.x_ld;
  const T* dy = (const T*)A.dy + row * A.dy_ld;
  const float mean = A.mean[row], rstd = A.rstd[row];
  float sums[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < A.cols; c += blockDim.x) {
    float g = to_f(dy[c]);
    if (A.w) g *= to_f(((const W*)A.w)[c]);
    sums[0] += g;
    sums[1] = fmaf(g, (to_f(x[c]) - mean) * rstd, sums[1]);
  }
  row_sum(sums, blockDim.x, 0);
  const float mg = sums[0] / (float)A.cols, mgx = sums[1] / (float)A.cols;
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

template <typename W>
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* __restrict__ partial,
                                                         int64_t rows, int64_t cols, W* dw, W* db) {
  column_join<W>(partial, rows, cols, dw, db, blockIdx.x);
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
  const int64_t b = kFeatSMs * (cols <= 256 ? 4 : 2);
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
  } else if (tpr <= 32 && A.rows >= 4096) {
    norm_forward_rows_kernel<T, W, VEC, 4>
        <<<(unsigned)ceil_div(A.rows, 128 / tpr * 4), 128, 0, st>>>(A);
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

template <typename T, typename W, int VEC, int R, bool PARAMS>
static int norm_backward_run(const NormArgs& A, int grid, int threads, cudaStream_t st) {
  // The ring, or afterwards the slots' sums.
  const int slots = A.tpr < 32 ? threads / 32 : threads / A.tpr;
  size_t smem = PARAMS && A.tpr < threads ? (size_t)slots * 2 * A.cols * sizeof(float) : 0;
  if constexpr (VEC > 1) {
    smem = std::max<size_t>(smem, (size_t)(kNormAhead<R> + 1) * R * 2 * threads * 16);
    constexpr auto kernel = norm_backward_kernel<T, W, VEC, R, PARAMS>;
    // The ring of the widest block; with the static part, 48 KB need no opt-in.
    constexpr int kMost = (kNormAhead<R> + 1) * R * 2 * 512 * 16;
    if (smem > 40 * 1024) GPB_TRY(allow_smem<kernel>(kMost));
    kernel<<<grid, threads, smem, st>>>(A);
  } else {
    norm_backward_scalar_kernel<T, W, R, PARAMS><<<grid, threads, smem, st>>>(A);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, typename W, int VEC, bool PARAMS>
static int norm_backward_vec(NormArgs A, int* blocks, cudaStream_t st, bool* done) {
  // 16 columns per thread in vectors, 8 otherwise (registers). A row takes as few threads as that
  // allows, but a warp before a second vector.
  constexpr int kMaxR = VEC == 1 ? 8 : 16 / VEC;
  const int64_t nvec = ceil_div(A.cols, VEC);
  int tpr = 1, r = 1;
  while (tpr < 32 && tpr < nvec) tpr <<= 1;
  while (r < kMaxR && (int64_t)tpr * r < nvec) r <<= 1;
  while (tpr < 512 && (int64_t)tpr * r < nvec) tpr <<= 1;
  *done = (int64_t)tpr * r >= nvec;
  if (!*done) return GPB_OK;
  A.tpr = tpr;
  const int threads = tpr > 256 ? tpr : 256;
  const int grid = (int)std::min<int64_t>(*blocks, ceil_div(A.rows, threads / tpr));
  *blocks = grid;
  switch (r) {
    case 1: return norm_backward_run<T, W, VEC, 1, PARAMS>(A, grid, threads, st);
    case 2: return norm_backward_run<T, W, VEC, 2 <= kMaxR ? 2 : kMaxR, PARAMS>(A, grid, threads, st);
    case 4: return norm_backward_run<T, W, VEC, 4 <= kMaxR ? 4 : kMaxR, PARAMS>(A, grid, threads, st);
    default: return norm_backward_run<T, W, VEC, kMaxR, PARAMS>(A, grid, threads, st);
  }
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
    norm_join_kernel<W><<<(unsigned)ceil_div(2 * (int64_t)A.cols, 32), 1024, 0, st>>>(
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
