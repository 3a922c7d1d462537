// Layer norm over the columns of a row-major [rows][cols] block, forward and backward.
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w,  xhat = (x - mean) rstd,  dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum_rows dy xhat,  db = sum_rows dy
// Everything is held in fp32 and rounded once, to the output's type. The variance is the second
// pass over the row's registers (no E[x^2] - mean^2 cancellation). dw and db are summed in a fixed
// order (per block in row order, then over blocks), so results repeat bit for bit.
//
// A row belongs to TPR threads (a power of two: part of a warp, or the block), each of which keeps
// R vectors of VEC elements in registers: x and dy are read once and dx is written once. HBM bound where
// there are many rows: 1M x 16 fp32 (136 MB with the statistics) 21.7 us, 16384 x 4096 bf16 (268 MB) 54 us,
// its backward pass (403 MB) 85 us with the join of dw and db. A few rows cost their launch.
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
// square root cost 30 instructions a row). The estimate of 0 is infinity and that of infinity 0: they
// are the results, and a step from them would be NaN.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  return v > 0.f && r > 0.f ? fmaf(fmaf(-0.5f * v * r, r, 0.5f), r, r) : r;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows in flight per thread in the rings below: what two resident blocks' rings have room for.
template <int R>
constexpr int kNormAhead = R >= 4 ? 2 : 4;
constexpr int kNormScalarAhead = 2;

// Shared memory of one unaligned row: its 16-byte blocks as they lie, the ones it only partly fills
// included. (A block that holds any of a row's bytes is inside the allocation that holds the row.)
__host__ __device__ constexpr int norm_slot_bytes(int cols, int es) {
  return (cols * es + 15 + 15) / 16 * 16;
}
template <typename T>
__device__ __forceinline__ void norm_copy_row(const T* p, int cols, char* slot, int lane, int tpr) {
  const char* first = reinterpret_cast<const char*>((uintptr_t)p & ~(uintptr_t)15);
  const int blocks = (int)(((uintptr_t)(p + cols) - (uintptr_t)first + 15) >> 4);
  const uint32_t dst = smem_addr(slot);
  for (int v = lane; v < blocks; v += tpr) copy16(dst + 16 * v, first + 16 * v);
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

// A row per TPR threads, R single elements each (unaligned rows, when they are few).
template <typename T, typename W, int R>
__global__ void __launch_bounds__(512) norm_forward_kernel(const NormArgs A) {
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < A.rows;
  const T* x = (const T*)A.x + (live ? row : 0) * A.x_ld;
  float v[R], s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = r * tpr + lane;
    v[r] = live && c < A.cols ? to_f(x[c]) : 0.f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) s[0] += v[r];
  row_sum(s, tpr, 0);
  const float inv = 1.f / (float)A.cols, mean = s[0] * inv;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    v[r] -= mean;
    q[0] = r * tpr + lane < A.cols ? fmaf(v[r], v[r], q[0]) : q[0];
  }
  row_sum(q, tpr, 1);
  const float rstd = inv_sqrt(fmaf(q[0], inv, A.eps));
  if (!live) return;
  if (lane == 0) {
    if (A.mean) A.mean[row] = mean;
    if (A.rstd) A.rstd[row] = rstd;
  }
  T* y = (T*)A.out + row * A.out_ld;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = r * tpr + lane;
    if (c >= A.cols) break;
    float o = v[r] * rstd;
    if (A.w) o *= to_f(((const W*)A.w)[c]);
    if (A.b) o += to_f(((const W*)A.b)[c]);
    y[c] = from_f<T>(o);
  }
}

// A row per TPR threads, R 16-byte vectors each, kept as they came (half the registers of their fp32
// values, so twice the rows in flight: those loads are what the kernel's rate depends on) and
// converted in each of the three passes.
template <typename T, typename W, int VEC, int R>
__global__ void __launch_bounds__(512) norm_forward_vec_kernel(const NormArgs A) {
  constexpr int P = VEC / 2;
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < A.rows;
  const int c0 = lane * VEC, dc = tpr * VEC;
  const T* x = (const T*)A.x + (live ? row : 0) * A.x_ld + c0;
  const T* tag = nullptr;
  uint4 raw[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    raw[r] = live && c0 + r * dc < A.cols ? *reinterpret_cast<const uint4*>(x + r * dc)
                                          : make_uint4(0, 0, 0, 0);
  const float inv = 1.f / (float)A.cols;
  float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float2 v[P];
    unpack16(raw[r], v, tag);
#pragma unroll
    for (int i = 0; i < P; ++i) s2 = __fadd2_rn(s2, v[i]);
  }
  float s[1] = {s2.x + s2.y};
  row_sum(s, tpr, 0);
  const float mean = s[0] * inv;
  const float2 neg_mean = make_float2(-mean, -mean);
  float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (c0 + r * dc < A.cols) {
      float2 v[P];
      unpack16(raw[r], v, tag);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 d = __fadd2_rn(v[i], neg_mean);
        q2 = __ffma2_rn(d, d, q2);
      }
    }
  }
  float q[1] = {q2.x + q2.y};
  row_sum(q, tpr, 1);
  const float rstd = inv_sqrt(fmaf(q[0], inv, A.eps));
  if (!live) return;
  if (lane == 0) {
    if (A.mean) A.mean[row] = mean;
    if (A.rstd) A.rstd[row] = rstd;
  }
  T* y = (T*)A.out + row * A.out_ld + c0;
  const float2 scale = make_float2(rstd, rstd);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = c0 + r * dc;
    if (c >= A.cols) break;
    float2 v[P];
    unpack16(raw[r], v, tag);
    float w[VEC], b[VEC];
    if (A.w) load_vec<W, VEC>((const W*)A.w + c, w);
    if (A.b) load_vec<W, VEC>((const W*)A.b + c, b);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      v[i] = __fmul2_rn(__fadd2_rn(v[i], neg_mean), scale);
      if (A.w) v[i] = __fmul2_rn(v[i], make_float2(w[2 * i], w[2 * i + 1]));
      if (A.b) v[i] = __fadd2_rn(v[i], make_float2(b[2 * i], b[2 * i + 1]));
    }
    *reinterpret_cast<uint4*>(y + r * dc) = pack16(v, tag);
  }
}

// Many unaligned rows: a fixed number of blocks walks them, copied to shared memory as they lie
// kNormScalarAhead rows ahead (60000 x 777 bf16: 180 us with single-element loads, 103 us). Aligned
// rows do not gain from such a ring: its blocks are too few for the two reductions of a row.
template <typename T, typename W, int R>
__global__ void __launch_bounds__(512) norm_forward_ring_kernel(const NormArgs A) {
  extern __shared__ __align__(16) char norm_ring[];
  constexpr int SLOTS = kNormScalarAhead + 1;
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr, group = threadIdx.x / tpr;
  const int64_t step = (int64_t)gridDim.x * groups;
  const int slot_bytes = norm_slot_bytes(A.cols, sizeof(T));
  char* ring = norm_ring + group * SLOTS * slot_bytes;
  auto fetch = [&](int64_t row, int s) {
    if (row < A.rows)
      norm_copy_row((const T*)A.x + row * A.x_ld, A.cols, ring + s * slot_bytes, lane, tpr);
    copy_commit();
  };
  const int64_t first = (int64_t)blockIdx.x * groups + group;
#pragma unroll
  for (int s = 0; s < kNormScalarAhead; ++s) fetch(first + s * step, s);
  const float inv = 1.f / (float)A.cols;
  int at = 0;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < A.rows;
    copy_wait<kNormScalarAhead - 1>();
    // Every thread's copies of this row are in, and every thread is done with the row before.
    if (tpr > 32)
      __syncthreads();
    else
      __syncwarp();
    fetch(row + kNormScalarAhead * step, at == 0 ? SLOTS - 1 : at - 1);
    const T* xg = (const T*)A.x + (live ? row : 0) * A.x_ld;
    const T* x = reinterpret_cast<const T*>(ring + at * slot_bytes + ((uintptr_t)xg & 15));
    float v[R], s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = r * tpr + lane;
      v[r] = live && c < A.cols ? to_f(x[c]) : 0.f;
      s[0] += v[r];
    }
    row_sum(s, tpr, 0);
    const float mean = s[0] * inv;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r] -= mean;
      q[0] = r * tpr + lane < A.cols ? fmaf(v[r], v[r], q[0]) : q[0];
    }
    row_sum(q, tpr, 1);
    const float rstd = inv_sqrt(fmaf(q[0], inv, A.eps));
    if (live) {
      if (lane == 0) {
        if (A.mean) A.mean[row] = mean;
        if (A.rstd) A.rstd[row] = rstd;
      }
      T* y = (T*)A.out + row * A.out_ld;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int c = r * tpr + lane;
        if (c >= A.cols) break;
        float o = v[r] * rstd;
        if (A.w) o *= to_f(((const W*)A.w)[c]);
        if (A.b) o += to_f(((const W*)A.b)[c]);
        y[c] = from_f<T>(o);
      }
    }
    at = at + 1 == SLOTS ? 0 : at + 1;
  }
  copy_wait<0>();
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
    const float scale = rstd, shift = -mean;
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
        // Subtracted first: x rstd - mean rstd would lose |mean| rstd 2^-24 in rows far from zero.
        xh[r][i] = __fmul2_rn(__fadd2_rn(xh[r][i], shift2), scale2);
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

// The same for rows that are not 16-byte aligned (an odd width, say): rows are copied to shared memory
// kNormScalarAhead ahead (norm_copy_row) and their elements read from there, one per lane. Loads of
// single elements leave too few bytes in flight: 60000 x 777 bf16 took 339 us, now 190 us.
template <typename T, typename W, int R, bool PARAMS>
__global__ void __launch_bounds__(512) norm_backward_scalar_kernel(const NormArgs A) {
  extern __shared__ __align__(16) float row_sums[];  // the ring, then [slots][2][cols]
  constexpr int SLOTS = kNormScalarAhead + 1;
  const int tpr = A.tpr;
  const int lane = threadIdx.x & (tpr - 1);
  const int groups = blockDim.x / tpr, group = threadIdx.x / tpr;
  const int slot_bytes = norm_slot_bytes(A.cols, sizeof(T));
  char* ring = reinterpret_cast<char*>(row_sums) + (int64_t)group * SLOTS * 2 * slot_bytes;
  const int64_t step = (int64_t)gridDim.x * groups;
  auto fetch = [&](int64_t row, int s) {
    if (row < A.rows) {
      norm_copy_row((const T*)A.x + row * A.x_ld, A.cols, ring + (2 * s) * slot_bytes, lane, tpr);
      norm_copy_row((const T*)A.dy + row * A.dy_ld, A.cols, ring + (2 * s + 1) * slot_bytes, lane, tpr);
    }
    copy_commit();
  };
  float dw[R][1], db[R][1];
#pragma unroll
  for (int r = 0; r < R; ++r) dw[r][0] = db[r][0] = 0.f;
  const int64_t row_first = (int64_t)blockIdx.x * groups + group;
#pragma unroll
  for (int s = 0; s < kNormScalarAhead; ++s) fetch(row_first + s * step, s);
  int flip = 0, at = 0;
  const float inv = 1.f / (float)A.cols;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < A.rows;
    copy_wait<kNormScalarAhead - 1>();
    // Every thread's copies of this row are in, and every thread is done with the row before.
    if (tpr > 32)
      __syncthreads();
    else
      __syncwarp();
    fetch(row + kNormScalarAhead * step, at == 0 ? SLOTS - 1 : at - 1);
    const int64_t rr = live ? row : 0;
    const T* xg = (const T*)A.x + rr * A.x_ld;
    const T* dg = (const T*)A.dy + rr * A.dy_ld;
    const T* x = reinterpret_cast<const T*>(ring + (2 * at) * slot_bytes + ((uintptr_t)xg & 15));
    const T* dy = reinterpret_cast<const T*>(ring + (2 * at + 1) * slot_bytes + ((uintptr_t)dg & 15));
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
    at = at + 1 == SLOTS ? 0 : at + 1;
  }
  copy_wait<0>();
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

// dw and db partial sums of rows too wide for the above: a thread owns VEC columns and walks a range
// of rows (blockIdx.y).
template <typename T, int VEC>
__global__ void __launch_bounds__(128) norm_params_wide_kernel(const NormArgs A) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * VEC;
  if (c >= A.cols) return;
  const int64_t per = (A.rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per;
  const int64_t r1 = r0 + per < A.rows ? r0 + per : A.rows;
  float dw[VEC], db[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) dw[i] = db[i] = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    float g[VEC], x[VEC];
    load_vec<T, VEC>((const T*)A.dy + r * A.dy_ld + c, g);
    load_vec<T, VEC>((const T*)A.x + r * A.x_ld + c, x);
    const float mean = A.mean[r], rstd = A.rstd[r];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      dw[i] = fmaf(g[i], (x[i] - mean) * rstd, dw[i]);
      db[i] += g[i];
    }
  }
  float* part = A.partial + (int64_t)blockIdx.y * 2 * A.cols + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    part[i] = dw[i];
    part[A.cols + i] = db[i];
  }
}

template <typename W>
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* __restrict__ partial,
                                                         int64_t rows, int64_t cols, W* dw, W* db) {
  column_join<W>(partial, rows, cols, dw, db, blockIdx.x);
}

// ------------------------------------------------------------------ host
// Threads per row and vectors per thread for `nvec` vectors. With many rows a row takes as few threads
// as it can (a warp first, then max_r vectors per thread): its loads are in flight together and
// fewer barriers join it. With few rows the widest spread answers soonest. Returns the vectors per
// thread, or 0 when the row does not fit 512 threads with max_r vectors each.
static int norm_shape(int64_t nvec, int max_r, int64_t rows, int* tpr) {
  const bool few = rows < 4 * kFeatSMs;
  int t = 1, r = 1;
  while (t < 32 && t < nvec) t <<= 1;
  if (!few)
    while (r < max_r && (int64_t)t * r < nvec) r <<= 1;
  while (t < 512 && (int64_t)t * r < nvec) t <<= 1;
  while (r < max_r && (int64_t)t * r < nvec) r <<= 1;
  *tpr = t;
  return (int64_t)t * r >= nvec ? r : 0;
}

// Blocks of the backward pass (each writes one partial row of 2 cols sums), a function of the sizes
// alone so that the workspace query and the launch agree.
static int norm_blocks(int64_t rows, int64_t cols) {
  const int64_t b = kFeatSMs * (cols <= 256 ? 4 : 2);
  return (int)(b < rows ? b : (rows > 0 ? rows : 1));
}

template <typename T, typename W, int R>
static int norm_forward_ring(const NormArgs& A, cudaStream_t st) {
  const int threads = A.tpr > 256 ? A.tpr : 256;
  const int groups = threads / A.tpr;
  const size_t smem = (size_t)groups * (kNormScalarAhead + 1) * norm_slot_bytes(A.cols, sizeof(T));
  constexpr auto kernel = norm_forward_ring_kernel<T, W, R>;
  if (smem > 40 * 1024) GPB_TRY(allow_smem<kernel>(200 * 1024));
  const int64_t grid = std::min<int64_t>(ceil_div(A.rows, groups), 4 * kFeatSMs);
  kernel<<<(unsigned)grid, threads, smem, st>>>(A);
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, typename W, int VEC, int R>
static void norm_forward_run(const NormArgs& A, cudaStream_t st) {
  const int threads = A.tpr > 128 ? A.tpr : 128;
  const unsigned grid = (unsigned)ceil_div(A.rows, threads / A.tpr);
  if constexpr (VEC > 1)
    norm_forward_vec_kernel<T, W, VEC, R><<<grid, threads, 0, st>>>(A);
  else
    norm_forward_kernel<T, W, R><<<grid, threads, 0, st>>>(A);
}

template <typename T, typename W, int VEC>
static int norm_forward_launch(NormArgs A, cudaStream_t st) {
  constexpr int kMaxR = 32 / VEC;
  int tpr = 1;
  const int64_t nvec = ceil_div(A.cols, VEC);
  const int r = norm_shape(nvec, kMaxR, A.rows, &tpr);
  A.tpr = tpr;
  if constexpr (VEC == 1) {
    // The ring: many rows of at most 16 elements per thread.
    int ring_tpr = 1;
    const int ring_r = norm_shape(nvec, 16, A.rows, &ring_tpr);
    if (nvec > 16 && A.rows >= 4 * kFeatSMs && ring_r) {
      A.tpr = ring_tpr;
      switch (ring_r) {
        case 1: return norm_forward_ring<T, W, 1>(A, st);
        case 2: return norm_forward_ring<T, W, 2>(A, st);
        case 4: return norm_forward_ring<T, W, 4>(A, st);
        case 8: return norm_forward_ring<T, W, 8>(A, st);
        default: return norm_forward_ring<T, W, 16>(A, st);
      }
    }
  }
  if (r == 0) {
    norm_forward_wide_kernel<T, W><<<(unsigned)A.rows, 1024, 0, st>>>(A);
  } else if (r == 1 && tpr <= 32 && A.rows >= 4096) {
    norm_forward_rows_kernel<T, W, VEC, 4>
        <<<(unsigned)ceil_div(A.rows, 128 / tpr * 4), 128, 0, st>>>(A);
  } else {
    switch (r) {
      case 1: norm_forward_run<T, W, VEC, 1>(A, st); break;
      case 2: norm_forward_run<T, W, VEC, 2>(A, st); break;
      case 4: norm_forward_run<T, W, VEC, 4>(A, st); break;
      case 8: norm_forward_run<T, W, VEC, 8 < kMaxR ? 8 : kMaxR>(A, st); break;
      case 16: norm_forward_run<T, W, VEC, 16 < kMaxR ? 16 : kMaxR>(A, st); break;
      default: norm_forward_run<T, W, VEC, kMaxR>(A, st);
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
    constexpr auto kernel = norm_backward_scalar_kernel<T, W, R, PARAMS>;
    smem = std::max<size_t>(smem, (size_t)(threads / A.tpr) * (kNormScalarAhead + 1) * 2 *
                                      norm_slot_bytes(A.cols, sizeof(T)));
    if (smem > 40 * 1024) GPB_TRY(allow_smem<kernel>(200 * 1024));
    kernel<<<grid, threads, smem, st>>>(A);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T, typename W, int VEC, bool PARAMS>
static int norm_backward_vec(NormArgs A, int* blocks, cudaStream_t st, bool* done) {
  // 16 columns per thread, 32 of 16 bits without the weight gradients (registers, and the ring's shared
  // memory). A row takes as few threads as that allows, but a warp before a second vector.
  constexpr int kMaxR = (PARAMS || VEC == 1 || sizeof(T) == 4 ? 16 : 32) / VEC;
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
    case 8: return norm_backward_run<T, W, VEC, 8 <= kMaxR ? 8 : kMaxR, PARAMS>(A, grid, threads, st);
    default: return norm_backward_run<T, W, VEC, kMaxR, PARAMS>(A, grid, threads, st);
  }
}

template <typename T, typename W, int VEC>
static int norm_backward_launch(NormArgs A, W* dw, W* db, cudaStream_t st) {
  const bool params = dw || db;
  int blocks = norm_blocks(A.rows, A.cols);
  bool done = false;
  if (params) GPB_TRY((norm_backward_vec<T, W, VEC, true>(A, &blocks, st, &done)));
  if (!done) {
    // The parameter sums read x and dy before dx may overwrite them in place.
    if (params) {
      blocks = (int)std::min<int64_t>(blocks, ceil_div(A.rows, 16));
      norm_params_wide_kernel<T, VEC>
          <<<dim3((unsigned)ceil_div(A.cols, 128 * VEC), blocks), 128, 0, st>>>(A);
      GPB_CHECK_CUDA(cudaGetLastError());
    }
    int unused = norm_blocks(A.rows, A.cols);
    if (A.out) GPB_TRY((norm_backward_vec<T, W, VEC, false>(A, &unused, st, &done)));
    if (A.out && !done) {
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
                  !overlaps(block_extent(out_dev, rows, cols, out_ld, es),
                            block_extent(x_dev, rows, cols, x_ld, es)),
              GPB_ERR_INVALID, "out overlaps x (in place needs the same pointer and stride)");
  {
    // The statistics are written while rows, weight and bias are still read.
    const Extent used[] = {block_extent(out_dev, rows, cols, out_ld, es),
                           block_extent(x_dev, rows, cols, x_ld, es), flat_extent(weight_dev, cols * ps),
                           flat_extent(bias_dev, cols * ps)};
    const Extent mean = flat_extent(mean_dev, rows * 4), rstd = flat_extent(rstd_dev, rows * 4);
    for (const Extent& u : used)
      GPB_REQUIRE(!overlaps(mean, u) && !overlaps(rstd, u), GPB_ERR_INVALID,
                  "mean or rstd overlaps another argument");
    GPB_REQUIRE(!overlaps(mean, rstd), GPB_ERR_INVALID, "mean and rstd overlap");
    for (int i = 2; i < 4; ++i)
      GPB_REQUIRE(!overlaps(used[0], used[i]), GPB_ERR_INVALID, "out overlaps weight or bias");
  }
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
  GPB_REQUIRE(elem_aligned(dweight_dev, ps) && elem_aligned(dbias_dev, ps), GPB_ERR_INVALID,
              "pointer is not aligned to its element type");
  if (rows == 0) {
    GPB_DEVICE_SCOPE(device);
    if (dweight_dev) GPB_CHECK_CUDA(cudaMemsetAsync(dweight_dev, 0, cols * ps, (cudaStream_t)stream));
    if (dbias_dev) GPB_CHECK_CUDA(cudaMemsetAsync(dbias_dev, 0, cols * ps, (cudaStream_t)stream));
    return GPB_OK;
  }
  GPB_REQUIRE(dx_dev || params, GPB_ERR_INVALID, "no output was asked for");
  GPB_REQUIRE(dout_dev && x_dev && mean_dev && rstd_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(dout_ld >= cols && x_ld >= cols && (!dx_dev || dx_ld >= cols), GPB_ERR_INVALID,
              "leading dimension below the %lld columns", (long long)cols);
  GPB_REQUIRE(elem_aligned(dx_dev, es) && elem_aligned(dout_dev, es) && elem_aligned(x_dev, es) &&
                  elem_aligned(weight_dev, ps) && elem_aligned(mean_dev, 4) &&
                  elem_aligned(rstd_dev, 4),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const Extent dx = block_extent(dx_dev, rows, cols, dx_ld, es),
               dout = block_extent(dout_dev, rows, cols, dout_ld, es),
               x = block_extent(x_dev, rows, cols, x_ld, es), weight = flat_extent(weight_dev, cols * ps),
               mean = flat_extent(mean_dev, rows * 4), rstd = flat_extent(rstd_dev, rows * 4);
  GPB_REQUIRE((dx_dev == dout_dev && dx_ld == dout_ld) || !overlaps(dx, dout),
              GPB_ERR_INVALID, "dx overlaps dout (in place needs the same pointer and stride)");
  GPB_REQUIRE((dx_dev == x_dev && dx_ld == x_ld) || !overlaps(dx, x),
              GPB_ERR_INVALID, "dx overlaps x (in place needs the same pointer and stride)");
  GPB_REQUIRE(!overlaps(dx, weight) && !overlaps(dx, mean) && !overlaps(dx, rstd), GPB_ERR_INVALID,
              "dx overlaps weight, mean or rstd");
  if (params) {
    const int64_t need = (int64_t)norm_blocks(rows, cols) * 2 * cols * (int64_t)sizeof(float);
    GPB_REQUIRE(workspace_dev && workspace_bytes >= need, GPB_ERR_INVALID,
                "the weight gradients need a workspace of %lld bytes, got %lld", (long long)need,
                (long long)(workspace_dev ? workspace_bytes : 0));
    GPB_REQUIRE(aligned16(workspace_dev), GPB_ERR_INVALID, "workspace is not 16-byte aligned");
    const Extent in[] = {dout, x, weight, mean, rstd};
    const Extent out[] = {dx, flat_extent(dweight_dev, cols * ps), flat_extent(dbias_dev, cols * ps),
                          flat_extent(workspace_dev, need)};
    for (int o = 1; o < 4; ++o) {
      for (const Extent& i : in)
        GPB_REQUIRE(!overlaps(out[o], i), GPB_ERR_INVALID,
                    "dweight, dbias or the workspace overlaps an input");
      for (int q = 0; q < o; ++q)
        GPB_REQUIRE(!overlaps(out[o], out[q]), GPB_ERR_INVALID,
                    "two outputs (or an output and the workspace) overlap");
    }
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
