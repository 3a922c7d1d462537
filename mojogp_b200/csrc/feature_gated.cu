// Gated projection unit: both projections, the activation and the product in one kernel.
//   gate = x Wg' + bg,  up = x Wu' + bu,  out = act(gate) * up
// x [rows][inner], Wg and Wu [outer][inner], row-major; out [rows][outer].
// Backward, with gate and up recomputed (they are never stored):
//   dgate = dout up act'(gate),  dup = dout act(gate)
//   dx = dgate Wg + dup Wu,  dWg = dgate' x,  dWu = dup' x,  dbg, dbu = column sums
// Sums are held in fp32. dgate and dup are rounded once to the element type, as operands of the
// three products that follow (fp32 inputs keep them in fp32).
#include <algorithm>
#include <cmath>

#include "features.cuh"

namespace gpb {

enum GatedAct : int32_t { ACT_SILU = 0, ACT_GELU = 1, ACT_SIGMOID = 2, ACT_TANH = 3 };

// act(z) and act'(z). Silu z s(z), gelu z Phi(z), with s the logistic function and Phi the normal
// distribution function (exact erf form).
__device__ __forceinline__ void gated_act(int act, float z, float& value, float& slope) {
  if (act == ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678f * z);
    value = z * cdf;
    slope = fmaf(z * 0.39894228f, expf(-0.5f * z * z), cdf);
  } else if (act == ACT_TANH) {
    value = tanhf(z);
    slope = fmaf(-value, value, 1.f);
  } else {
    const float s = 1.f / (1.f + expf(-z));
    if (act == ACT_SIGMOID) {
      value = s;
      slope = s * (1.f - s);
    } else {
      value = z * s;
      slope = s * fmaf(z, 1.f - s, 1.f);
    }
  }
}

struct GatedArgs {
  const void* x;
  const void* wg;
  const void* wu;
  const void* bg;
  const void* bu;
  const void* dout;
  void* out;   // forward
  void* dg;    // backward: [rows][outer] operands of the products
  void* du;
  int64_t x_ld, w_ld, out_ld, dout_ld;
  int64_t rows, inner, outer;
  int32_t act;
};

constexpr int kTile = 64, kTileK = 16;

// One 64 x 64 tile of both projections per block, 256 threads x 4 x 4 values each; BACK writes dgate
// and dup instead of the product.
template <typename T, bool BACK>
__global__ void __launch_bounds__(256) gated_simt_kernel(const GatedArgs A) {
  __shared__ float xs[kTileK][kTile + 4], gs[kTileK][kTile + 4], us[kTileK][kTile + 4];
  const int64_t tiles_n = (A.outer + kTile - 1) / kTile;
  const int64_t m0 = (blockIdx.x / tiles_n) * kTile, n0 = (blockIdx.x % tiles_n) * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float g[4][4] = {}, u[4][4] = {};
  for (int64_t k0 = 0; k0 < A.inner; k0 += kTileK) {
    for (int q = threadIdx.x; q < kTile * kTileK; q += 256) {
      const int r = q / kTileK, k = q % kTileK;
      const bool kin = k0 + k < A.inner;
      xs[k][r] = kin && m0 + r < A.rows ? to_f(((const T*)A.x)[(m0 + r) * A.x_ld + k0 + k]) : 0.f;
      const bool in = kin && n0 + r < A.outer;
      const int64_t wi = (n0 + r) * A.w_ld + k0 + k;
      gs[k][r] = in ? to_f(((const T*)A.wg)[wi]) : 0.f;
      us[k][r] = in ? to_f(((const T*)A.wu)[wi]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileK; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = xs[k][ty * 4 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[i][j] = fmaf(a, gs[k][tx * 4 + j], g[i][j]);
          u[i][j] = fmaf(a, us[k][tx * 4 + j], u[i][j]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= A.rows) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= A.outer) break;
      const float gate = g[i][j] + (A.bg ? to_f(((const T*)A.bg)[n]) : 0.f);
      const float up = u[i][j] + (A.bu ? to_f(((const T*)A.bu)[n]) : 0.f);
      float value, slope;
      gated_act(A.act, gate, value, slope);
      if constexpr (BACK) {
        const float dy = to_f(((const T*)A.dout)[m * A.dout_ld + n]);
        ((T*)A.dg)[m * A.outer + n] = from_f<T>(dy * up * slope);
        ((T*)A.du)[m * A.outer + n] = from_f<T>(dy * value);
      } else {
        ((T*)A.out)[m * A.out_ld + n] = from_f<T>(value * up);
      }
    }
  }
}

// C [m][n] = sum over terms and k of A_t(m, k) B_t(k, n), any strides; blockIdx.z = a range of k whose
// fp32 partial sums go to `partial` (one range: C is written directly).
struct MmTerm {
  const void* a;
  const void* b;
};
struct MmArgs {
  MmTerm term[2];
  int32_t terms;
  int64_t a_m, a_k, b_k, b_n;
  int64_t M, N, K;
  void* c;
  int64_t c_ld;
  float* partial;
  int64_t k_per;
};

template <typename T>
__global__ void __launch_bounds__(256) mm_simt_kernel(const MmArgs A) {
  __shared__ float as[kTileK][kTile + 4], bs[kTileK][kTile + 4];
  const int64_t tiles_n = (A.N + kTile - 1) / kTile;
  const int64_t m0 = (blockIdx.x / tiles_n) * kTile, n0 = (blockIdx.x % tiles_n) * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t kb = blockIdx.z * A.k_per;
  const int64_t ke = kb + A.k_per < A.K ? kb + A.k_per : A.K;
  float c[4][4] = {};
  for (int t = 0; t < A.terms; ++t) {
    const T* a = (const T*)A.term[t].a;
    const T* b = (const T*)A.term[t].b;
    for (int64_t k0 = kb; k0 < ke; k0 += kTileK) {
      for (int q = threadIdx.x; q < kTile * kTileK; q += 256) {
        // Neighbouring threads along the unit stride of each operand.
        const int ar = A.a_k == 1 ? q / kTileK : q % kTile, ak = A.a_k == 1 ? q % kTileK : q / kTile;
        const int br = A.b_k == 1 ? q / kTileK : q % kTile, bk = A.b_k == 1 ? q % kTileK : q / kTile;
        as[ak][ar] = k0 + ak < ke && m0 + ar < A.M
                         ? to_f(a[(m0 + ar) * A.a_m + (k0 + ak) * A.a_k]) : 0.f;
        bs[bk][br] = k0 + bk < ke && n0 + br < A.N
                         ? to_f(b[(k0 + bk) * A.b_k + (n0 + br) * A.b_n]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kTileK; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            c[i][j] = fmaf(as[k][ty * 4 + i], bs[k][tx * 4 + j], c[i][j]);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= A.M) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= A.N) break;
      if (gridDim.z == 1)
        ((T*)A.c)[m * A.c_ld + n] = from_f<T>(c[i][j]);
      else
        A.partial[(blockIdx.z * A.M + m) * A.N + n] = c[i][j];
    }
  }
}

// C = sum of the ranges' partial sums, in range order.
template <typename T>
__global__ void __launch_bounds__(256) mm_join_kernel(const float* __restrict__ partial, int ranges,
                                                      int64_t M, int64_t N, T* c, int64_t c_ld) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= M * N) return;
  float s = 0.f;
  for (int r = 0; r < ranges; ++r) s += partial[r * M * N + e];
  c[(e / N) * c_ld + e % N] = from_f<T>(s);
}

// Column sums of dgate and dup (blockIdx.y picks one): 32 columns x 8 row lanes per block, rows in
// ranges over blockIdx.z, joined by gated_bias_join.
template <typename T>
__global__ void __launch_bounds__(256) gated_bias_kernel(const T* dg, const T* du, int64_t rows,
                                                         int64_t outer, float* partial) {
  __shared__ float sums[8][33];
  const T* d = blockIdx.y == 0 ? dg : du;
  const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int part = threadIdx.x >> 5;
  const int64_t per = (rows + gridDim.z - 1) / gridDim.z;
  const int64_t r0 = blockIdx.z * per, r1 = r0 + per < rows ? r0 + per : rows;
  float s = 0.f;
  if (c < outer)
    for (int64_t r = r0 + part; r < r1; r += 8) s += to_f(d[r * outer + c]);
  sums[part][threadIdx.x & 31] = s;
  __syncthreads();
  if (part == 0 && c < outer) {
    for (int q = 1; q < 8; ++q) s += sums[q][threadIdx.x & 31];
    partial[((int64_t)blockIdx.z * 2 + blockIdx.y) * outer + c] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) gated_bias_join(const float* partial, int ranges,
                                                       int64_t outer, T* dbg, T* dbu) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= 2 * outer) return;
  float s = 0.f;
  for (int r = 0; r < ranges; ++r) s += partial[r * 2 * outer + e];
  T* dst = e < outer ? dbg : dbu;
  if (dst) dst[e < outer ? e : e - outer] = from_f<T>(s);
}

// ------------------------------------------------------------------ host
// Workspace of the backward pass: dgate | dup | partial sums.
struct GatedPlan {
  int64_t dg = 0, du = 0, partial = 0, total = 0;
  int ranges_w = 1;  // ranges of rows for dWg and dWu
  int ranges_b = 1;  // ranges of rows for the biases
};

static GatedPlan gated_plan(int64_t rows, int64_t inner, int64_t outer, int32_t dtype, bool backward) {
  GatedPlan P;
  if (!backward) return P;
  const int64_t op = round_up(rows * outer * dtype_bytes(dtype), 256);
  P.dg = 0;
  P.du = op;
  P.partial = 2 * op;
  const int64_t tiles = ceil_div(outer, kTile) * ceil_div(inner, kTile);
  int64_t r = ceil_div(4 * kFeatSMs, tiles);
  r = std::min<int64_t>(r, ceil_div(rows, 256));
  P.ranges_w = (int)std::max<int64_t>(1, r);
  P.ranges_b = (int)std::max<int64_t>(
      1, std::min<int64_t>(ceil_div(4 * kFeatSMs, ceil_div(outer, 32)), ceil_div(rows, 256)));
  const int64_t pw = P.ranges_w > 1 ? P.ranges_w * outer * inner : 0;
  P.total = P.partial + round_up(std::max<int64_t>(pw, P.ranges_b * 2 * outer) * 4, 256);
  return P;
}

template <typename T>
static int gated_forward(const GatedArgs& A, cudaStream_t st) {
  const int64_t grid = ceil_div(A.rows, kTile) * ceil_div(A.outer, kTile);
  gated_simt_kernel<T, false><<<(unsigned)grid, 256, 0, st>>>(A);
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}

template <typename T>
static int mm_launch(MmArgs M, int ranges, cudaStream_t st) {
  const int64_t grid = ceil_div(M.M, kTile) * ceil_div(M.N, kTile);
  M.k_per = round_up(ceil_div(M.K, ranges), kTileK);
  ranges = (int)ceil_div(M.K, M.k_per);
  mm_simt_kernel<T><<<dim3((unsigned)grid, 1, ranges), 256, 0, st>>>(M);
  GPB_CHECK_CUDA(cudaGetLastError());
  if (ranges > 1) {
    mm_join_kernel<T><<<(unsigned)ceil_div(M.M * M.N, 256), 256, 0, st>>>(M.partial, ranges, M.M,
                                                                         M.N, (T*)M.c, M.c_ld);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

struct GatedGrads {
  void* dx;
  int64_t dx_ld;
  void* dwg;
  void* dwu;
  int64_t dw_ld;
  void* dbg;
  void* dbu;
};

template <typename T>
static int gated_backward(GatedArgs A, const GatedGrads& G, char* ws, const GatedPlan& P,
                          cudaStream_t st) {
  A.dg = ws + P.dg;
  A.du = ws + P.du;
  float* partial = (float*)(ws + P.partial);
  const int64_t grid = ceil_div(A.rows, kTile) * ceil_div(A.outer, kTile);
  gated_simt_kernel<T, true><<<(unsigned)grid, 256, 0, st>>>(A);
  GPB_CHECK_CUDA(cudaGetLastError());
  if (G.dx) {
    MmArgs M{};
    M.term[0] = {A.dg, A.wg};
    M.term[1] = {A.du, A.wu};
    M.terms = 2;
    M.a_m = A.outer;
    M.a_k = 1;
    M.b_k = A.w_ld;
    M.b_n = 1;
    M.M = A.rows;
    M.N = A.inner;
    M.K = A.outer;
    M.c = G.dx;
    M.c_ld = G.dx_ld;
    GPB_TRY(mm_launch<T>(M, 1, st));
  }
  for (int h = 0; h < 2; ++h) {
    void* dw = h == 0 ? G.dwg : G.dwu;
    if (!dw) continue;
    MmArgs M{};
    M.term[0] = {h == 0 ? A.dg : A.du, A.x};
    M.terms = 1;
    M.a_m = 1;
    M.a_k = A.outer;
    M.b_k = A.x_ld;
    M.b_n = 1;
    M.M = A.outer;
    M.N = A.inner;
    M.K = A.rows;
    M.c = dw;
    M.c_ld = G.dw_ld;
    M.partial = partial;
    GPB_TRY(mm_launch<T>(M, P.ranges_w, st));
  }
  if (G.dbg || G.dbu) {
    gated_bias_kernel<T><<<dim3((unsigned)ceil_div(A.outer, 32), 2, P.ranges_b), 256, 0, st>>>(
        (const T*)A.dg, (const T*)A.du, A.rows, A.outer, partial);
    GPB_CHECK_CUDA(cudaGetLastError());
    gated_bias_join<T><<<(unsigned)ceil_div(2 * A.outer, 256), 256, 0, st>>>(
        partial, P.ranges_b, A.outer, (T*)G.dbg, (T*)G.dbu);
    GPB_CHECK_CUDA(cudaGetLastError());
  }
  return GPB_OK;
}

static int gated_check(int32_t dtype, int64_t rows, int64_t inner, int64_t outer) {
  GPB_REQUIRE(dtype_ok(dtype), GPB_ERR_INVALID, "unknown element type %d", dtype);
  GPB_REQUIRE(rows >= 0 && inner >= 1 && outer >= 1, GPB_ERR_INVALID,
              "gated unit needs rows >= 0, inner >= 1 and outer >= 1, got %lld, %lld, %lld",
              (long long)rows, (long long)inner, (long long)outer);
  GPB_REQUIRE(rows < ((int64_t)1 << 31) && inner <= (1 << 20) && outer <= (1 << 20),
              GPB_ERR_INVALID, "gated unit sizes %lld, %lld, %lld are too large (2^31, 2^20, 2^20)",
              (long long)rows, (long long)inner, (long long)outer);
  GPB_REQUIRE(rows * std::max(inner, outer) <= ((int64_t)1 << 40), GPB_ERR_INVALID,
              "gated unit of %lld rows is too large", (long long)rows);
  return GPB_OK;
}

}  // namespace gpb

using namespace gpb;

extern "C" {

int gpb_gated_unit_workspace(int32_t dtype, int64_t rows, int64_t inner, int64_t outer,
                             int32_t backward, int64_t* bytes_out) {
  clear_error();
  GPB_REQUIRE(bytes_out, GPB_ERR_INVALID, "null output");
  GPB_TRY(gated_check(dtype, rows, inner, outer));
  *bytes_out = gated_plan(rows, inner, outer, dtype, backward != 0).total;
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
  const int64_t ob = span_bytes(rows, outer, out_ld, es), wb = span_bytes(outer, inner, w_ld, es);
  GPB_REQUIRE(!overlaps(out_dev, ob, x_dev, span_bytes(rows, inner, x_ld, es)) &&
                  !overlaps(out_dev, ob, w_gate_dev, wb) && !overlaps(out_dev, ob, w_up_dev, wb) &&
                  !overlaps(out_dev, ob, b_gate_dev, outer * es) &&
                  !overlaps(out_dev, ob, b_up_dev, outer * es),
              GPB_ERR_INVALID, "out overlaps an input");
  const GatedPlan P = gated_plan(rows, inner, outer, dtype, false);
  GPB_REQUIRE(P.total == 0 || (workspace_dev && workspace_bytes >= P.total), GPB_ERR_INVALID,
              "gated unit needs a workspace of %lld bytes, got %lld", (long long)P.total,
              (long long)(workspace_dev ? workspace_bytes : 0));
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
  switch (dtype) {
    case GPB_DTYPE_F32: return gated_forward<float>(A, st);
    case GPB_DTYPE_F16: return gated_forward<__half>(A, st);
    default: return gated_forward<__nv_bfloat16>(A, st);
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
  GPB_REQUIRE(dx_dev || dw_gate_dev || dw_up_dev || db_gate_dev || db_up_dev, GPB_ERR_INVALID,
              "no output was asked for");
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
  GPB_REQUIRE(dout_dev && x_dev && w_gate_dev && w_up_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(x_ld >= inner && w_ld >= inner && dout_ld >= outer, GPB_ERR_INVALID,
              "leading dimension below the column count");
  GPB_REQUIRE(elem_aligned(dout_dev, es) && elem_aligned(x_dev, es) &&
                  elem_aligned(w_gate_dev, es) && elem_aligned(w_up_dev, es) &&
                  elem_aligned(b_gate_dev, es) && elem_aligned(b_up_dev, es),
              GPB_ERR_INVALID, "pointer is not aligned to its element type");
  const GatedPlan P = gated_plan(rows, inner, outer, dtype, true);
  GPB_REQUIRE(workspace_dev && workspace_bytes >= P.total, GPB_ERR_INVALID,
              "the backward pass needs a workspace of %lld bytes, got %lld", (long long)P.total,
              (long long)(workspace_dev ? workspace_bytes : 0));
  GPB_REQUIRE(((uintptr_t)workspace_dev & 15u) == 0, GPB_ERR_INVALID,
              "workspace is not 16-byte aligned");
  {
    // Outputs and the workspace are written while inputs are still read: none may share memory.
    const int64_t wb = span_bytes(outer, inner, w_ld, es), bb = outer * es;
    const struct { const void* p; int64_t n; } in[] = {
        {dout_dev, span_bytes(rows, outer, dout_ld, es)}, {x_dev, span_bytes(rows, inner, x_ld, es)},
        {w_gate_dev, wb}, {w_up_dev, wb}, {b_gate_dev, bb}, {b_up_dev, bb}};
    const int64_t dwb = span_bytes(outer, inner, dw_ld, es);
    const struct { const void* p; int64_t n; } out[] = {
        {dx_dev, span_bytes(rows, inner, dx_ld, es)}, {dw_gate_dev, dwb}, {dw_up_dev, dwb},
        {db_gate_dev, bb}, {db_up_dev, bb}, {workspace_dev, P.total}};
    for (int o = 0; o < 6; ++o) {
      for (const auto& i : in)
        GPB_REQUIRE(!overlaps(out[o].p, out[o].n, i.p, i.n), GPB_ERR_INVALID,
                    "an output or the workspace overlaps an input");
      for (int q = 0; q < o; ++q)
        GPB_REQUIRE(!overlaps(out[o].p, out[o].n, out[q].p, out[q].n), GPB_ERR_INVALID,
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
  switch (dtype) {
    case GPB_DTYPE_F32: return gated_backward<float>(A, G, (char*)workspace_dev, P, st);
    case GPB_DTYPE_F16: return gated_backward<__half>(A, G, (char*)workspace_dev, P, st);
    default: return gated_backward<__nv_bfloat16>(A, G, (char*)workspace_dev, P, st);
  }
}

}  // extern "C"
