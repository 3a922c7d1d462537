// Gradient of the kernel's bilinear form with respect to the training inputs:
//   out_i = d/dx_i sum_c a_c' K b_c = sum_j G_ij d1 k(x_i, x_j),
//   G_ij = sum_c (a_ci b_cj + b_ci a_cj)
// (d1: with respect to the first argument; the second argument's part is folded in by symmetry).
// With a = [alpha | u_c], b = [alpha | P^-1 z_c] of a BBMM step it is the NLL's gradient by the
// inputs, which a learned feature map's backward pass starts from.
//
// One stationary leaf (with or without a scale node): d1 k = -psi (x_i - x_j) / l^2 with
// psi = -2 dk/ds, s the scaled squared distance. Two kernels:
//   few columns (up to 4): G_ij on the CUDA cores, two rows per thread;
//   more: G = [a | b]' [b | a] is a product of depth 32, formed on the tensor cores (bf16 planes, six
//     products, fp32-accurate) into TMEM while the CUDA cores run psi and the sums over j. On the CUDA
//     cores G was 32 of the 74 FMAs of a pair: 2.0 ms at 20000 points in 8 dimensions with 16 columns,
//     0.71 ms here (Matern-5/2; the FP32 pipe alone would take 0.61).
// Both work on fp32 pairs (FFMA2), split the columns of a row tile over a cluster of 8 blocks and
// join through distributed shared memory, in block order: no workspace (a captured graph owns
// nothing) and no atomics.
//
// Differences are taken between prescaled inputs x / l, except for Matern-1/2: its psi grows as 1 / r,
// so the direction of near pairs counts, which rounding x / l would lose; there the raw inputs are
// subtracted and the difference scaled.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "gated_gemm.cuh"
#include "provider.cuh"

namespace gpb {

namespace cg = cooperative_groups;

struct InputGradArgs {
  const float* X;    // [n][d]
  const float* a;    // [cols][n]
  const float* b;
  float* out;        // [n][d]
  int64_t n;
  int32_t d, nd, cols, accumulate;
  float power;       // RQ: alpha + 1
  int32_t clamp12;   // Matern-1/2 ARD bounds its exponent
  int32_t dims[GPB_MAX_DIM];
  float scale[GPB_MAX_DIM];      // of the inputs; 0 past nd
  float out_scale[GPB_MAX_DIM];  // of the sums
  int* err;                  // the provider's device error word
};

// psi of the leaf at squared distance s of inputs scaled by 1 / l and the leaf's own constant (which
// leaves one multiplication between a square root and an exponential), without the factor that
// provider_input_gradient folds into out_scale; the same clamps as the leaf's value and parameter
// gradients (kernel_program.cuh).
template <int LEAF>
__device__ __forceinline__ float pair_psi(float s, const InputGradArgs& A) {
  if constexpr (LEAF == GPB_KERNEL_RBF) {  // s / (2 ln 2)
    return ex2_approx(-s);
  } else if constexpr (LEAF == GPB_KERNEL_RQ) {  // s / (2 alpha)
    return ex2_approx(-A.power * lg2_approx(1.f + s));
  } else {
    const float ss = fmaxf(s, 1e-20f);
    float rinv;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(rinv) : "f"(ss));
    const float r = ss * rinv;
    if constexpr (LEAF == GPB_KERNEL_MATERN12) {
      const float x = r * -kLog2e;
      return ex2_approx(A.clamp12 ? fmaxf(x, -20.f * kLog2e) : x) * rinv;
    } else {
      const float e = ex2_approx(fmaxf(r * -kLog2e, -20.f * kLog2e));  // 3 s, 5 s
      return LEAF == GPB_KERNEL_MATERN32 ? e : fmaf(r, e, e);
    }
  }
}

constexpr int kIgThreads = 128;
constexpr int kIgTile = 32;     // columns staged per step
constexpr int kIgCluster = 8;   // blocks along the columns of one row tile

// x (a row's coordinates as pairs) minus a column's, scaled where the inputs are raw.
template <int LEAF, int D2>
__device__ __forceinline__ void ig_diff(const InputGradArgs& A, const float2 (&x)[D2],
                                        const float2* col, float2 (&diff)[D2]) {
#pragma unroll
  for (int q = 0; q < D2; ++q) {
    const float2 c = col[q];  // negated
    diff[q] = __fadd2_rn(x[q], c);
    if constexpr (LEAF == GPB_KERNEL_MATERN12)
      diff[q] = __fmul2_rn(diff[q], make_float2(A.scale[2 * q], A.scale[2 * q + 1]));
  }
}

// Input coordinate f of point i as the kernels subtract it.
template <int LEAF>
__device__ __forceinline__ float ig_coord(const InputGradArgs& A, int64_t i, int f) {
  if (i >= A.n || f >= A.nd) return 0.f;
  const float x = A.X[i * A.d + A.dims[f]];
  return LEAF == GPB_KERNEL_MATERN12 ? x : x * A.scale[f];
}

// Adds the cluster's sums [parts][rows][D] in block order and writes rows congruent to this block's
// rank. Every thread of the cluster takes part.
template <int D, int PARTS>
__device__ __forceinline__ void ig_join(const InputGradArgs& A, float* sums, int rows, int64_t row0) {
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int lr = blockIdx.y + threadIdx.x * kIgCluster; lr < rows; lr += blockDim.x * kIgCluster) {
    const int64_t i = row0 + lr;
    if (i >= A.n) continue;
    float* o = A.out + i * A.d;
    if (!A.accumulate)
      for (int q = 0; q < A.d; ++q) o[q] = 0.f;
    for (int q = 0; q < A.nd; ++q) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kIgCluster; ++k) {
        const float* remote = cluster.map_shared_rank(sums, k);
        for (int p = 0; p < PARTS; ++p) s += remote[(p * rows + lr) * D + q];
      }
      o[A.dims[q]] -= s * A.out_scale[q];
    }
  }
  cluster.sync();
}

// Up to 4 right-hand-side pairs; D input dims (an even number, padded with zeros), R rows per thread.
template <int LEAF, int D, int R>
__global__ void __cluster_dims__(1, kIgCluster, 1) __launch_bounds__(kIgThreads)
    input_gradient_kernel(const __grid_constant__ InputGradArgs A) {
  constexpr int T = 4, D2 = D / 2;
  constexpr int W = D + 2 * T;
  __shared__ __align__(16) float tile[2][kIgTile * W];
  extern __shared__ float sums[];  // [R * kIgThreads][D]
  const int64_t row0 = (int64_t)blockIdx.x * (kIgThreads * R) + threadIdx.x;
  float2 xi[R][D2], acc[R][D2];
  float2 ai[R][T / 2], bi[R][T / 2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = row0 + r * kIgThreads;
#pragma unroll
    for (int q = 0; q < D2; ++q) {
      xi[r][q] = make_float2(ig_coord<LEAF>(A, i, 2 * q), ig_coord<LEAF>(A, i, 2 * q + 1));
      acc[r][q] = make_float2(0.f, 0.f);
    }
    auto rhs = [&](const float* v, int c) { return i < A.n && c < A.cols ? v[c * A.n + i] : 0.f; };
#pragma unroll
    for (int c = 0; c < T / 2; ++c) {
      ai[r][c] = make_float2(rhs(A.a, 2 * c), rhs(A.a, 2 * c + 1));
      bi[r][c] = make_float2(rhs(A.b, 2 * c), rhs(A.b, 2 * c + 1));
    }
  }
  const int64_t tiles = (A.n + kIgTile - 1) / kIgTile;
  // Columns past n carry zero a and b, so they add psi * 0.
  constexpr int PER = (kIgTile * W + kIgThreads - 1) / kIgThreads;
  float next[PER];
  auto load = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int q = threadIdx.x + u * kIgThreads;
      const int f = q / kIgTile;
      const int64_t j = t * kIgTile + q % kIgTile;
      float v = 0.f;
      if (t < tiles && j < A.n) {
        if (f < D)
          v = -ig_coord<LEAF>(A, j, f);
        else if (f < D + T)
          v = f - D < A.cols ? A.b[(int64_t)(f - D) * A.n + j] : 0.f;
        else if (f < W)
          v = f - D - T < A.cols ? A.a[(int64_t)(f - D - T) * A.n + j] : 0.f;
      }
      next[u] = v;
    }
  };
  load(blockIdx.y);
  int buf = 0;
  for (int64_t t = blockIdx.y; t < tiles; t += kIgCluster, buf ^= 1) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int q = threadIdx.x + u * kIgThreads;
      if (q < kIgTile * W) tile[buf][(q % kIgTile) * W + q / kIgTile] = next[u];
    }
    __syncthreads();
    load(t + kIgCluster);
    // The tile's own sums first: fewer terms per running sum, half the rounding error.
    float2 part[R][D2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < D2; ++q) part[r][q] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int j = 0; j < kIgTile; ++j) {
      const float2* col = reinterpret_cast<const float2*>(tile[buf] + j * W);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 diff[D2], s = make_float2(0.f, 0.f), g = make_float2(0.f, 0.f);
        ig_diff<LEAF, D2>(A, xi[r], col, diff);
#pragma unroll
        for (int q = 0; q < D2; ++q) s = __ffma2_rn(diff[q], diff[q], s);
#pragma unroll
        for (int c = 0; c < T / 2; ++c) {
          g = __ffma2_rn(ai[r][c], col[D2 + c], g);
          g = __ffma2_rn(bi[r][c], col[D2 + T / 2 + c], g);
        }
        const float w = (g.x + g.y) * pair_psi<LEAF>(s.x + s.y, A);
        const float2 w2 = make_float2(w, w);
#pragma unroll
        for (int q = 0; q < D2; ++q) part[r][q] = __ffma2_rn(w2, diff[q], part[r][q]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < D2; ++q) acc[r][q] = __fadd2_rn(acc[r][q], part[r][q]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int q = 0; q < D2; ++q) {
      sums[(r * kIgThreads + threadIdx.x) * D + 2 * q] = acc[r][q].x;
      sums[(r * kIgThreads + threadIdx.x) * D + 2 * q + 1] = acc[r][q].y;
    }
  ig_join<D, 1>(A, sums, R * kIgThreads, (int64_t)blockIdx.x * (kIgThreads * R));
}

// ------------------------------------------------------- tensor-core G
// 8 warps run the pairs (TMEM lane quadrant = warp % 4, two warps share a tile's columns), 4 warps
// split a and b of the next 128 columns into bf16 planes and issue its 12 MMAs; two tiles are in
// flight, each with its own operand planes, coordinates and 128 TMEM columns.
constexpr int kIgcThreads = 384;
constexpr int kIgcCols = 128;
constexpr int kIgcPlane = 128 * 32 * 2;       // bytes: 128 points, depth 32, 16-bit
constexpr int kIgcOperand = 3 * kIgcPlane;

// Byte offset of (point p, depth 8 q) in a plane: 8-point x 16-byte core matrices, points adjacent
// at 128 bytes, depth at 2048.
__device__ __forceinline__ int igc_offset(int p, int q) {
  return q * 2048 + (p >> 3) * 128 + (p & 7) * 16;
}

// Depth 8 q .. 8 q + 7 of one point: right-hand sides 8 (q % 2) .. of `lo` (q < 2) or `hi`, which
// point at the point's column 0. Each value is the exact sum of three bf16 parts (rounded to nearest);
// one past bf16's range or not finite makes its products NaN.
__device__ __forceinline__ void igc_split(const InputGradArgs& A, const float* lo, const float* hi,
                                          bool in, int q, int p, char* planes) {
  const int c0 = (q & 1) * 8;
  const float* v = (q < 2 ? lo : hi) + c0 * A.n;
  float2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i].x = in && c0 + 2 * i < A.cols ? *v : 0.f;
    v += A.n;
    x[i].y = in && c0 + 2 * i + 1 < A.cols ? *v : 0.f;
    v += A.n;
  }
  char* dst = planes + igc_offset(p, q);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = gg_part<__nv_bfloat16>(x[i]);
    *reinterpret_cast<uint4*>(dst + k * kIgcPlane) = make_uint4(h[0], h[1], h[2], h[3]);
  }
}

__device__ __forceinline__ void igc_load(uint32_t addr, uint32_t (&r)[16]) { tmem_ld16_async(addr, r); }
__device__ __forceinline__ void igc_load(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <int D>
struct IgcShape {
  static constexpr int kCoords = kIgcCols * D * 4;
  static constexpr int kSmem = 3 * kIgcOperand + 2 * kCoords;  // rows, two column tiles
  // The join's sums [2][128][D] reuse the column tiles.
  static_assert(2 * 128 * D * 4 <= 2 * kIgcOperand + 2 * kCoords, "join fits");
  static constexpr int kBlocks = D <= 8 ? 2 : 1;    // per SM (registers)
  static constexpr int kChunk = D <= 16 ? 16 : 4;   // columns per TMEM load
};

template <int LEAF, int D>
__global__ void __cluster_dims__(1, kIgCluster, 1)
    __launch_bounds__(kIgcThreads, IgcShape<D>::kBlocks)
        input_gradient_tc_kernel(const __grid_constant__ InputGradArgs A) {
  constexpr int D2 = D / 2, CH = IgcShape<D>::kChunk;
  extern __shared__ __align__(128) char ig_smem[];
  char* row_planes = ig_smem;
  char* col_planes = ig_smem + kIgcOperand;
  float* coords = reinterpret_cast<float*>(ig_smem + 3 * kIgcOperand);
  __shared__ __align__(8) uint64_t full[2], empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&full[s], 4 + 1);  // the producer warps and the MMAs' completion
      mbar_init(&empty[s], 8);
    }
    fence_barrier_init();
    failed = 0;
  }
  if (warp == 8) tmem_alloc(&tmem_base, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const int64_t row0 = (int64_t)blockIdx.x * 128;
  const int64_t tiles = (A.n + kIgcCols - 1) / kIgcCols;
  const int mine = blockIdx.y < tiles ? (int)((tiles - blockIdx.y + kIgCluster - 1) / kIgCluster) : 0;
  float2 acc[D2];
#pragma unroll
  for (int q = 0; q < D2; ++q) acc[q] = make_float2(0.f, 0.f);

  if (warp >= 8) {
    const int p = threadIdx.x - 256;
#pragma unroll 1
    for (int q = 0; q < 4; ++q)
      igc_split(A, A.a + row0 + p, A.b + row0 + p, row0 + p < A.n, q, p, row_planes);
    constexpr uint32_t idesc = gg_idesc(true, false, false, kIgcCols);
    bool ok = true;
    for (int t = 0; t < mine; ++t) {
      const int s = t & 1;
      const int64_t j = ((int64_t)blockIdx.y + (int64_t)t * kIgCluster) * kIgcCols + p;
      if (t >= 2) ok = mbar_wait_bounded(&empty[s], ((t >> 1) & 1) ^ 1);
      // The four warps stay together: a wait that ran out in one ends all of them.
      if (!ok) failed = 1;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (*(volatile int*)&failed) break;
      char* planes = col_planes + s * kIgcOperand;
#pragma unroll 1
      for (int q = 0; q < 4; ++q) igc_split(A, A.b + j, A.a + j, j < A.n, q, p, planes);
      float* x = coords + (s * kIgcCols + p) * D;
#pragma unroll 1
      for (int f = 0; f < D; ++f) x[f] = -ig_coord<LEAF>(A, j, f);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (threadIdx.x == 256) {
        tc_fence_after();
        const uint32_t d = tmem + s * kIgcCols;
        uint64_t da[3], db[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          da[k] = make_smem_desc(row_planes + k * kIgcPlane, 2048, 128);
          db[k] = make_smem_desc(planes + k * kIgcPlane, 2048, 128);
        }
        constexpr uint32_t next = 4096 >> 4;  // 16 deeper
        // Small products first: the accumulator truncates, and only the last two MMAs are large.
        gg_mma(d, da[2], db[0], idesc, 0);
        gg_mma(d, da[2] + next, db[0] + next, idesc, 1);
        gg_mma(d, da[1], db[1], idesc, 1);
        gg_mma(d, da[1] + next, db[1] + next, idesc, 1);
        gg_mma(d, da[0], db[2], idesc, 1);
        gg_mma(d, da[0] + next, db[2] + next, idesc, 1);
        gg_mma(d, da[1], db[0], idesc, 1);
        gg_mma(d, da[1] + next, db[0] + next, idesc, 1);
        gg_mma(d, da[0], db[1], idesc, 1);
        gg_mma(d, da[0] + next, db[1] + next, idesc, 1);
        gg_mma(d, da[0], db[0], idesc, 1);
        gg_mma(d, da[0] + next, db[0] + next, idesc, 1);
        mma_commit(&full[s]);
      }
    }
    if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
  } else {
    const int quad = warp & 3, half = warp >> 2;
    const int64_t i = row0 + quad * 32 + lane;
    float2 xi[D2];
#pragma unroll
    for (int q = 0; q < D2; ++q)
      xi[q] = make_float2(ig_coord<LEAF>(A, i, 2 * q), ig_coord<LEAF>(A, i, 2 * q + 1));
    bool ok = true;
    for (int t = 0; t < mine; ++t) {
      const int s = t & 1;
      ok = mbar_wait_bounded(&full[s], (t >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t g_addr = tmem + s * kIgcCols + ((uint32_t)quad << 21) + half * 64;
      const float* x = coords + (s * kIgcCols + half * 64) * D;
#pragma unroll 1
      for (int c = 0; c < 64; c += CH) {
        uint32_t g[CH];
        igc_load(g_addr + c, g);
        tmem_wait_ld();
        // These columns' own sums first: fewer terms per running sum, less rounding error.
        float2 part[D2];
#pragma unroll
        for (int q = 0; q < D2; ++q) part[q] = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          const float2* col = reinterpret_cast<const float2*>(x + (c + k) * D);
          float2 sq = make_float2(0.f, 0.f);
          if constexpr (D <= 16) {
            float2 diff[D2];
            ig_diff<LEAF, D2>(A, xi, col, diff);
#pragma unroll
            for (int q = 0; q < D2; ++q) sq = __ffma2_rn(diff[q], diff[q], sq);
            const float w = __uint_as_float(g[k]) * pair_psi<LEAF>(sq.x + sq.y, A);
            const float2 w2 = make_float2(w, w);
#pragma unroll
            for (int q = 0; q < D2; ++q) part[q] = __ffma2_rn(w2, diff[q], part[q]);
          } else {
            // The differences twice. At 64 dimensions a row, its sums and the differences are 192 registers (the
            // kernel spills 244 to 356 bytes even so: 20000 points, 16 columns 10 ms); 32 take the same path.
#pragma unroll
            for (int q = 0; q < D2; ++q) {
              float2 diff = __fadd2_rn(xi[q], col[q]);
              if constexpr (LEAF == GPB_KERNEL_MATERN12)
                diff = __fmul2_rn(diff, make_float2(A.scale[2 * q], A.scale[2 * q + 1]));
              sq = __ffma2_rn(diff, diff, sq);
            }
            const float w = __uint_as_float(g[k]) * pair_psi<LEAF>(sq.x + sq.y, A);
            const float2 w2 = make_float2(w, w);
#pragma unroll
            for (int q = 0; q < D2; ++q) {
              float2 diff = __fadd2_rn(xi[q], col[q]);
              if constexpr (LEAF == GPB_KERNEL_MATERN12)
                diff = __fmul2_rn(diff, make_float2(A.scale[2 * q], A.scale[2 * q + 1]));
              acc[q] = __ffma2_rn(w2, diff, acc[q]);
            }
          }
        }
        if constexpr (D <= 16)
#pragma unroll
          for (int q = 0; q < D2; ++q) acc[q] = __fadd2_rn(acc[q], part[q]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 256);
  float* sums = reinterpret_cast<float*>(col_planes);  // [2][128][D]
  if (warp < 8) {
    float* o = sums + ((warp >> 2) * 128 + (warp & 3) * 32 + lane) * D;
#pragma unroll
    for (int q = 0; q < D2; ++q) {
      o[2 * q] = acc[q].x;
      o[2 * q + 1] = acc[q].y;
    }
  }
  ig_join<D, 2>(A, sums, 128, row0);
}

// -------------------------------------------------------- any kernel tree
// d leaf / d xi scaled by `w`, added to g (length d).
__device__ __noinline__ void leaf_input_grad(const DevKernel& K, const LeafDesc& L, const float* xi,
                                             const float* xj, float w, float* g) {
  const float* p = K.params + L.pofs;
  const int nd = L.ndims;
  const int nl = L.ard ? nd : 1;
  if (is_stationary(L.type)) {
    float s = 0.f;
    for (int k = 0; k < nd; ++k) {
      const float dk = (xi[L.dims[k]] - xj[L.dims[k]]) / p[L.ard ? k : 0];
      s = fmaf(dk, dk, s);
    }
    const float r = sqrtf(fmaxf(s, 1e-20f));
    float psi;
    switch (L.type) {
      case GPB_KERNEL_RBF: psi = expf(-0.5f * s); break;
      case GPB_KERNEL_MATERN12: psi = expf(L.ard ? fmaxf(-r, -20.f) : -r) / r; break;
      case GPB_KERNEL_MATERN32: psi = 3.f * expf(fmaxf(-1.7320508075688772f * r, -20.f)); break;
      case GPB_KERNEL_MATERN52: {
        const float r5 = 2.23606797749979f * r;
        psi = (5.f / 3.f) * (1.f + r5) * expf(fmaxf(-r5, -20.f));
        break;
      }
      default: psi = powf(1.f + s / (2.f * p[nl]), -p[nl] - 1.f);
    }
    const float os = p[L.type == GPB_KERNEL_RQ ? nl + 1 : nl];
    for (int k = 0; k < nd; ++k) {
      const float l = p[L.ard ? k : 0];
      g[L.dims[k]] -= w * os * psi * ((xi[L.dims[k]] - xj[L.dims[k]]) / l) / l;
    }
  } else if (L.type == GPB_KERNEL_PERIODIC) {
    const float f = 3.14159265358979f / p[nl];
    const float kval = leaf_eval(K, L, xi, xj, nullptr);
    for (int k = 0; k < nd; ++k) {
      float sn, cs;
      sincosf(f * (xi[L.dims[k]] - xj[L.dims[k]]), &sn, &cs);
      g[L.dims[k]] -= w * kval * 4.f * f * sn * cs / p[L.ard ? k : 0];
    }
  } else if (L.type == GPB_KERNEL_LINEAR) {
    for (int k = 0; k < nd; ++k) g[L.dims[k]] += w * p[nl] * p[L.ard ? k : 0] * xj[L.dims[k]];
  } else {  // polynomial: iso [degree, offset, os], ARD [var..., degree, offset, os]
    const int base_i = L.ard ? nd : 0;
    const int degree = (int)lrintf(p[base_i]);
    float base = p[base_i + 1];
    for (int k = 0; k < nd; ++k) {
      const float prod = xi[L.dims[k]] * xj[L.dims[k]];
      base = L.ard ? fmaf(p[k], prod, base) : base + prod;
    }
    float slope = p[base_i + 2] * (float)degree;
    for (int q = 1; q < degree; ++q) slope *= base;
    for (int k = 0; k < nd; ++k) g[L.dims[k]] += w * slope * (L.ard ? p[k] : 1.f) * xj[L.dims[k]];
  }
}

// One warp per row, lanes over the columns; leaf adjoints by reverse accumulation over the program.
__global__ void __launch_bounds__(128) input_gradient_tree_kernel(
    const float* __restrict__ X, int64_t n, int d, const float* __restrict__ a,
    const float* __restrict__ b, int cols, int accumulate, float* __restrict__ out,
    const __grid_constant__ DevKernel K) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= n) return;
  float xi[GPB_MAX_DIM], xj[GPB_MAX_DIM], g[GPB_MAX_DIM];
  for (int k = 0; k < d; ++k) {
    xi[k] = X[i * d + k];
    g[k] = 0.f;
  }
  for (int64_t j = lane; j < n; j += 32) {
    float w = 0.f;
    for (int c = 0; c < cols; ++c) {
      w = fmaf(a[c * n + i], b[c * n + j], w);
      w = fmaf(b[c * n + i], a[c * n + j], w);
    }
    for (int k = 0; k < d; ++k) xj[k] = X[j * d + k];
    float val[GPB_MAX_NODES], adj[GPB_MAX_NODES];
    int child0[GPB_MAX_NODES], child1[GPB_MAX_NODES], stack[GPB_MAX_NODES];
    int sp = 0;
    for (int q = 0; q < K.nnodes; ++q) {
      const int op = K.node_op[q];
      child0[q] = child1[q] = -1;
      adj[q] = 0.f;
      if (op == GPB_NODE_LEAF) {
        val[q] = leaf_eval(K, K.leaf[K.node_arg[q]], xi, xj, nullptr);
      } else if (op == GPB_NODE_SCALE) {
        child0[q] = stack[--sp];
        val[q] = K.params[K.node_arg[q]] * val[child0[q]];
      } else {
        child1[q] = stack[--sp];
        child0[q] = stack[--sp];
        val[q] = op == GPB_NODE_SUM ? val[child0[q]] + val[child1[q]]
                                    : val[child0[q]] * val[child1[q]];
      }
      stack[sp++] = q;
    }
    adj[K.nnodes - 1] = w;
    for (int q = K.nnodes - 1; q >= 0; --q) {
      const int op = K.node_op[q];
      if (op == GPB_NODE_LEAF) {
        leaf_input_grad(K, K.leaf[K.node_arg[q]], xi, xj, adj[q], g);
      } else if (op == GPB_NODE_SCALE) {
        adj[child0[q]] += adj[q] * K.params[K.node_arg[q]];
      } else if (op == GPB_NODE_SUM) {
        adj[child0[q]] += adj[q];
        adj[child1[q]] += adj[q];
      } else {
        adj[child0[q]] += adj[q] * val[child1[q]];
        adj[child1[q]] += adj[q] * val[child0[q]];
      }
    }
  }
  for (int k = 0; k < d; ++k) {
    float s = g[k];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) out[i * d + k] = accumulate ? out[i * d + k] + s : s;
  }
}

// ------------------------------------------------------------------ host
template <int LEAF, int D>
static int launch_ig(InputGradArgs& A, cudaStream_t st) {
  if (A.cols > 4) {
    constexpr auto kernel = input_gradient_tc_kernel<LEAF, D>;
    GPB_TRY(allow_smem<kernel>(IgcShape<D>::kSmem));
    kernel<<<dim3((unsigned)ceil_div(A.n, 128), kIgCluster), kIgcThreads, IgcShape<D>::kSmem, st>>>(A);
  } else {
    constexpr int R = D <= 16 ? 2 : 1;  // a row's state is 2 D + 8 values
    constexpr int smem = R * kIgThreads * D * (int)sizeof(float);
    // The column tiles are static shared memory beside it: 50 KB in all at 64 dimensions.
    constexpr int tiles = 2 * kIgTile * (D + 8) * (int)sizeof(float);
    static_assert(smem + tiles <= 227 * 1024, "shared memory of a block");
    constexpr auto kernel = input_gradient_kernel<LEAF, D, R>;
    if constexpr (smem + tiles > 47 * 1024) GPB_TRY(allow_smem<kernel>(smem));
    kernel<<<dim3((unsigned)ceil_div(A.n, R * kIgThreads), kIgCluster), kIgThreads, smem, st>>>(A);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <int LEAF>
static int launch_ig_d(InputGradArgs& A, cudaStream_t st) {
  if (A.nd <= 2) return launch_ig<LEAF, 2>(A, st);
  if (A.nd <= 4) return launch_ig<LEAF, 4>(A, st);
  if (A.nd <= 8) return launch_ig<LEAF, 8>(A, st);
  if (A.nd <= 16) return launch_ig<LEAF, 16>(A, st);
  if (A.nd <= 32) return launch_ig<LEAF, 32>(A, st);
  return launch_ig<LEAF, 64>(A, st);
}

int provider_input_gradient(gpb_provider* p, float* out, const float* a, const float* b,
                            int64_t ncols, cudaStream_t st) {
  const DevKernel& K = p->dk;
  const bool one = K.nnodes == 1 || (K.nnodes == 2 && K.node_op[1] == GPB_NODE_SCALE);
  if (!one || !is_stationary(K.leaf[0].type)) {
    for (int64_t c = 0; c < ncols; c += 16) {
      input_gradient_tree_kernel<<<(unsigned)ceil_div(p->n, 4), 128, 0, st>>>(
          p->X_d, p->n, p->d, a + c * p->n, b + c * p->n, (int)std::min<int64_t>(16, ncols - c),
          c > 0, out, K);
      GPB_CHECK_CUDA(cudaGetLastError());
    }
    return GPB_OK;
  }
  const LeafDesc& L = K.leaf[0];
  const float* prm = K.params + L.pofs;
  const int nl = L.ard ? L.ndims : 1;
  InputGradArgs A{};
  A.X = p->X_d;
  A.out = out;
  A.n = p->n;
  A.d = p->d;
  A.nd = L.ndims;
  double os = L.type == GPB_KERNEL_RQ ? prm[nl + 1] : prm[nl];
  if (K.nnodes == 2) os *= K.params[K.node_arg[1]];
  // Input scale beyond 1 / l, and psi's constant factor.
  double c = 1.0, factor = 1.0;
  switch (L.type) {
    case GPB_KERNEL_RBF: c = std::sqrt(0.5 / std::log(2.0)); break;
    case GPB_KERNEL_MATERN32: c = std::sqrt(3.0), factor = 3.0; break;
    case GPB_KERNEL_MATERN52: c = std::sqrt(5.0), factor = 5.0 / 3.0; break;
    case GPB_KERNEL_RQ: c = std::sqrt(0.5 / (double)prm[nl]), A.power = prm[nl] + 1.f; break;
    default: break;
  }
  A.clamp12 = L.ard;
  A.err = p->err_d;
  for (int q = 0; q < L.ndims; ++q) {
    A.dims[q] = L.dims[q];
    const double l = prm[L.ard ? q : 0];
    A.scale[q] = (float)(c / l);
    A.out_scale[q] = (float)(os * factor / (c * l));
  }
  for (int64_t c = 0; c < ncols; c += 16) {
    A.a = a + c * p->n;
    A.b = b + c * p->n;
    A.cols = (int32_t)std::min<int64_t>(16, ncols - c);
    A.accumulate = c > 0;
    int s;
    switch (L.type) {
      case GPB_KERNEL_RBF: s = launch_ig_d<GPB_KERNEL_RBF>(A, st); break;
      case GPB_KERNEL_MATERN12: s = launch_ig_d<GPB_KERNEL_MATERN12>(A, st); break;
      case GPB_KERNEL_MATERN32: s = launch_ig_d<GPB_KERNEL_MATERN32>(A, st); break;
      case GPB_KERNEL_MATERN52: s = launch_ig_d<GPB_KERNEL_MATERN52>(A, st); break;
      default: s = launch_ig_d<GPB_KERNEL_RQ>(A, st);
    }
    GPB_TRY(s);
  }
  return GPB_OK;
}

}  // namespace gpb

using namespace gpb;

extern "C" int gpb_input_gradient(gpb_provider* p, float* out_dev, const float* a_dev,
                                  const float* b_dev, int64_t ncols, void* stream) {
  clear_error();
  GPB_REQUIRE(p && out_dev && a_dev && b_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(ncols >= 1, GPB_ERR_INVALID, "input gradient needs at least one column, got %lld",
              (long long)ncols);
  GPB_REQUIRE(elem_aligned(out_dev, 4) && elem_aligned(a_dev, 4) && elem_aligned(b_dev, 4),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const int64_t ob = p->n * p->d * 4, vb = p->n * ncols * 4;
  GPB_REQUIRE(!overlaps(out_dev, ob, a_dev, vb) && !overlaps(out_dev, ob, b_dev, vb) &&
                  !overlaps(out_dev, ob, p->X_d, ob),
              GPB_ERR_INVALID, "out overlaps an input");
  GPB_DEVICE_SCOPE(p->device);
  return provider_input_gradient(p, out_dev, a_dev, b_dev, ncols,
                                 stream ? (cudaStream_t)stream : p->stream);
}
