// Gradient of the kernel's bilinear form with respect to the training inputs:
//   out_i = d/dx_i sum_c a_c' K b_c = sum_j G_ij d1 k(x_i, x_j),
//   G_ij = sum_c (a_ci b_cj + b_ci a_cj)
// (d1: with respect to the first argument; the second argument's part is folded in by symmetry).
// With a = [alpha | u_c], b = [alpha | P^-1 z_c] of a BBMM step it is the NLL's gradient by the
// inputs, which a learned feature map's backward pass starts from.
//
// One stationary leaf (with or without a scale node): d1 k = -psi (x_i - x_j) / l^2 with
// psi = -2 dk/ds, s the scaled squared distance. Differences are taken between the raw inputs and
// scaled after: prescaled inputs would lose the direction of near pairs to their rounding, which
// Matern-1/2 does not damp. A thread owns two rows and a cluster of 8 blocks splits the columns of a
// row tile and joins through distributed shared memory, in block order: no workspace (a captured
// graph owns nothing) and no atomics.
#include <cooperative_groups.h>

#include <algorithm>

#include "features.cuh"
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
  float os, alpha;   // effective output scale, RQ alpha
  int32_t clamp12;   // Matern-1/2 ARD bounds its exponent
  int32_t dims[GPB_MAX_DIM];
  float inv_l[GPB_MAX_DIM];
};

// psi of the leaf at scaled squared distance s, without the output scale; the same clamps as the
// leaf's own value and parameter gradients (kernel_program.cuh).
template <int LEAF>
__device__ __forceinline__ float leaf_psi(float s, float alpha, int clamp12) {
  if constexpr (LEAF == GPB_KERNEL_RBF) {
    return ex2_approx(s * (-0.5f * kLog2e));
  } else if constexpr (LEAF == GPB_KERNEL_RQ) {
    const float base = 1.f + s / (2.f * alpha);
    return ex2_approx(-(alpha + 1.f) * lg2_approx(base));
  } else {
    const float ss = fmaxf(s, 1e-20f);
    const float rinv = rsqrtf(ss);
    const float r = ss * rinv;
    if constexpr (LEAF == GPB_KERNEL_MATERN12) {
      const float e = ex2_approx((clamp12 ? fmaxf(-r, -20.f) : -r) * kLog2e);
      return e * rinv;
    } else if constexpr (LEAF == GPB_KERNEL_MATERN32) {
      return 3.f * ex2_approx(fmaxf(-1.7320508075688772f * r, -20.f) * kLog2e);
    } else {
      const float r5 = 2.23606797749979f * r;
      return (5.f / 3.f) * (1.f + r5) * ex2_approx(fmaxf(-r5, -20.f) * kLog2e);
    }
  }
}

constexpr int kIgThreads = 128;
constexpr int kIgTile = 32;     // columns staged per step
constexpr int kIgCluster = 8;   // blocks along the columns of one row tile

// T right-hand-side pairs, D input dims (padded with zeros), R rows per thread.
template <int LEAF, int D, int T, int R>
__global__ void __cluster_dims__(1, kIgCluster, 1) __launch_bounds__(kIgThreads)
    input_gradient_kernel(const __grid_constant__ InputGradArgs A) {
  constexpr int W = (D + 2 * T + 3) / 4 * 4;
  __shared__ __align__(16) float tile[kIgTile * W];
  extern __shared__ float sums[];  // [R * kIgThreads][D]
  const int64_t row0 = (int64_t)blockIdx.x * (kIgThreads * R) + threadIdx.x;
  float xi[R][D], ai[R][T], bi[R][T], acc[R][D];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = row0 + r * kIgThreads;
    const bool in = i < A.n;
#pragma unroll
    for (int q = 0; q < D; ++q) {
      xi[r][q] = in && q < A.nd ? A.X[i * A.d + A.dims[q]] : 0.f;
      acc[r][q] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < T; ++c) {
      ai[r][c] = in && c < A.cols ? A.a[c * A.n + i] : 0.f;
      bi[r][c] = in && c < A.cols ? A.b[c * A.n + i] : 0.f;
    }
  }
  const int64_t tiles = (A.n + kIgTile - 1) / kIgTile;
  for (int64_t t = blockIdx.y; t < tiles; t += kIgCluster) {
    const int64_t j0 = t * kIgTile;
    __syncthreads();
    for (int q = threadIdx.x; q < kIgTile * (D + 2 * T); q += kIgThreads) {
      const int f = q / kIgTile, j = q % kIgTile;
      const bool in = j0 + j < A.n;
      float v = 0.f;
      if (f < D) {
        if (in && f < A.nd) v = A.X[(j0 + j) * A.d + A.dims[f]];
      } else if (f < D + T) {
        if (in && f - D < A.cols) v = A.a[(int64_t)(f - D) * A.n + j0 + j];
      } else {
        if (in && f - D - T < A.cols) v = A.b[(int64_t)(f - D - T) * A.n + j0 + j];
      }
      tile[j * W + f] = v;
    }
    __syncthreads();
    // Columns past n carry zero a and b, so their weight is 0 at whatever finite psi; none is
    // evaluated all the same.
    const int jn = (int)(A.n - j0 < kIgTile ? A.n - j0 : kIgTile);
    for (int j = 0; j < jn; ++j) {
      float col[W];
#pragma unroll
      for (int q = 0; q < W / 4; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(tile + j * W + 4 * q);
        col[4 * q] = v.x;
        col[4 * q + 1] = v.y;
        col[4 * q + 2] = v.z;
        col[4 * q + 3] = v.w;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float diff[D], s = 0.f, g = 0.f;
#pragma unroll
        for (int q = 0; q < D; ++q) {
          diff[q] = (xi[r][q] - col[q]) * A.inv_l[q];
          s = fmaf(diff[q], diff[q], s);
        }
#pragma unroll
        for (int c = 0; c < T; ++c) {
          g = fmaf(ai[r][c], col[D + T + c], g);
          g = fmaf(bi[r][c], col[D + c], g);
        }
        g *= leaf_psi<LEAF>(s, A.alpha, A.clamp12);
#pragma unroll
        for (int q = 0; q < D; ++q) acc[r][q] = fmaf(g, diff[q], acc[r][q]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int q = 0; q < D; ++q) sums[(r * kIgThreads + threadIdx.x) * D + q] = acc[r][q];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  // Each block of the cluster writes the rows congruent to its rank: one thread per row.
  for (int lr = blockIdx.y + threadIdx.x * kIgCluster; lr < R * kIgThreads;
       lr += kIgThreads * kIgCluster) {
    const int64_t i = (int64_t)blockIdx.x * (kIgThreads * R) + lr;
    if (i >= A.n) continue;
    float* o = A.out + i * A.d;
    if (!A.accumulate)
      for (int q = 0; q < A.d; ++q) o[q] = 0.f;
    for (int q = 0; q < A.nd; ++q) {
      float s = 0.f;
      for (int k = 0; k < kIgCluster; ++k) s += cluster.map_shared_rank(sums, k)[lr * D + q];
      o[A.dims[q]] -= s * A.os * A.inv_l[q];
    }
  }
  cluster.sync();
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
    float psi;
    switch (L.type) {
      case GPB_KERNEL_RBF: psi = leaf_psi<GPB_KERNEL_RBF>(s, 0.f, 0); break;
      case GPB_KERNEL_MATERN12: psi = leaf_psi<GPB_KERNEL_MATERN12>(s, 0.f, L.ard); break;
      case GPB_KERNEL_MATERN32: psi = leaf_psi<GPB_KERNEL_MATERN32>(s, 0.f, 0); break;
      case GPB_KERNEL_MATERN52: psi = leaf_psi<GPB_KERNEL_MATERN52>(s, 0.f, 0); break;
      default: psi = leaf_psi<GPB_KERNEL_RQ>(s, p[nl], 0);
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
template <int LEAF, int D, int T>
static int launch_ig(const InputGradArgs& A, cudaStream_t st) {
  // Two rows per thread where their state (2 D + 2 T values a row) fits the registers.
  constexpr int R = D <= 16 ? 2 : 1;
  const size_t smem = (size_t)R * kIgThreads * D * sizeof(float);
  const unsigned gx = (unsigned)ceil_div(A.n, R * kIgThreads);
  input_gradient_kernel<LEAF, D, T, R><<<dim3(gx, kIgCluster), kIgThreads, smem, st>>>(A);
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <int LEAF, int T>
static int launch_ig_d(const InputGradArgs& A, cudaStream_t st) {
  if (A.nd <= 1) return launch_ig<LEAF, 1, T>(A, st);
  if (A.nd <= 2) return launch_ig<LEAF, 2, T>(A, st);
  if (A.nd <= 4) return launch_ig<LEAF, 4, T>(A, st);
  if (A.nd <= 8) return launch_ig<LEAF, 8, T>(A, st);
  if (A.nd <= 16) return launch_ig<LEAF, 16, T>(A, st);
  if (A.nd <= 32) return launch_ig<LEAF, 32, T>(A, st);
  return launch_ig<LEAF, 64, T>(A, st);
}

template <int LEAF>
static int launch_ig_t(const InputGradArgs& A, cudaStream_t st) {
  return A.cols <= 4 ? launch_ig_d<LEAF, 4>(A, st) : launch_ig_d<LEAF, 16>(A, st);
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
  A.os = L.type == GPB_KERNEL_RQ ? prm[nl + 1] : prm[nl];
  A.alpha = L.type == GPB_KERNEL_RQ ? prm[nl] : 0.f;
  if (K.nnodes == 2) A.os *= K.params[K.node_arg[1]];
  A.clamp12 = L.ard;
  for (int q = 0; q < L.ndims; ++q) {
    A.dims[q] = L.dims[q];
    A.inv_l[q] = 1.f / prm[L.ard ? q : 0];
  }
  for (int64_t c = 0; c < ncols; c += 16) {
    A.a = a + c * p->n;
    A.b = b + c * p->n;
    A.cols = (int32_t)std::min<int64_t>(16, ncols - c);
    A.accumulate = c > 0;
    int s;
    switch (L.type) {
      case GPB_KERNEL_RBF: s = launch_ig_t<GPB_KERNEL_RBF>(A, st); break;
      case GPB_KERNEL_MATERN12: s = launch_ig_t<GPB_KERNEL_MATERN12>(A, st); break;
      case GPB_KERNEL_MATERN32: s = launch_ig_t<GPB_KERNEL_MATERN32>(A, st); break;
      case GPB_KERNEL_MATERN52: s = launch_ig_t<GPB_KERNEL_MATERN52>(A, st); break;
      default: s = launch_ig_t<GPB_KERNEL_RQ>(A, st);
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
