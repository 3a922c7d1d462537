// The gated unit's matrix products on the 5th-generation tensor cores (tcgen05, kind::f16).
//
// One persistent kernel, three products over 16-bit operands with fp32 accumulators in TMEM:
//   GG_PROJ  gate | up = x [Wg' | Wu']   tile 128 rows x (BN gate + BN up columns): both projections
//            of the same outputs share the x tile and one MMA, and the epilogue applies the
//            activation and the product (or, for the backward pass, forms dgate and dup);
//   GG_DX    dx = dgate Wg + dup Wu      one accumulation over two segments;
//   GG_DW    dWg = dgate' x, dWu = dup' x   the reduction runs over rows, which are split over CTAs
//            when the weight has few tiles (fp32 partial sums, joined in split order).
// x and the weights are read where they lie. A product whose reduction index is not the contiguous
// one takes its operand MN-major: the tensor core transposes, nothing is copied.
//
// fp32 inputs are exact sums of three bf16 planes (8 significant bits each), and
// a product keeps the six plane pairs above 2^-24 of it: hi hi apart from the five small ones, which
// have their own accumulator. The tensor core truncates where it adds, about 2^-26 of the accumulator
// per MMA, so after every kGgWindow blocks of the reduction the epilogue warps add both accumulators
// to registers in fp32 and the MMAs start again from zero.
//
// 10 warps: TMA producer, MMA issuer, 8 epilogue warps (TMEM lane quadrant = warp % 4, two warps
// share a quadrant's columns). Tiles move by cp.async.bulk.tensor into 128-byte-swizzled stages;
// accumulators are double-buffered so that a tile's epilogue runs under the next tile's MMAs. Every
// wait is bounded: one that runs out sets the module's error word and ends the role.
#pragma once

#include <cuda.h>

#include "features.cuh"
#include "tcgen05.cuh"

namespace gpb {

enum GatedAct : int32_t { ACT_SILU = 0, ACT_GELU = 1, ACT_SIGMOID = 2, ACT_TANH = 3 };

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(z) and, with SLOPE, act'(z), to about 2^-21. Silu is z s(z) with s the logistic function, gelu
// z Phi(z) with Phi the normal distribution function. An activation is one or two MUFU operations and
// some ten FMAs: with erfcf / expf / division and a load per bias the epilogue was instruction-bound
// (at 8192 x 1024 -> 4096, bf16, the backward projections took 315 us and take 162 us; the forward
// pass at 8192 x 2048 -> 8192 467 us, now 402 us).
template <bool SLOPE>
__device__ __forceinline__ void act_sigmoid(float z, float& value, float& slope) {
  value = rcp_approx(1.f + ex2_approx(-kLog2e * z));
  if constexpr (SLOPE) slope = fmaf(-value, value, value);
}
template <bool SLOPE>
__device__ __forceinline__ void act_silu(float z, float& value, float& slope) {
  const float s = rcp_approx(1.f + ex2_approx(-kLog2e * z));
  value = z * s;
  if constexpr (SLOPE) slope = fmaf(value, 1.f - s, s);
}
// tanh: 1 - 2 / (1 + e^2|z|), which cancels near 0; there z + z^3 Q(z^2), a degree-4 minimax fit on
// [0, 0.65] (3e-8).
template <bool SLOPE>
__device__ __forceinline__ void act_tanh(float z, float& value, float& slope) {
  const float a = fabsf(z), u = z * z;
  float q = fmaf(u, -0.00592442462220788f, 0.0208740234375f);
  q = fmaf(u, q, -0.05382389947772026f);
  q = fmaf(u, q, 0.13332584500312805f);
  q = fmaf(u, q, -0.333333283662796f);
  const float near = fmaf(z * u, q, z);
  const float far = fmaf(-2.f, rcp_approx(1.f + ex2_approx(2.f * kLog2e * a)), 1.f);
  value = a < 0.6f ? near : copysignf(far, z);
  if constexpr (SLOPE) slope = fmaf(-value, value, 1.f);
}
// Phi(-|z|) e^(z^2 / 2) is smooth in t = 1 / (1 + 0.3 |z|): a degree-8 minimax fit of relative error
// 1.5e-7 on |z| <= 14, fitted for this. The exponential serves the density in the slope too.
template <bool SLOPE>
__device__ __forceinline__ void act_gelu(float z, float& value, float& slope) {
  const float t = rcp_approx(fmaf(0.3f, fabsf(z), 1.f));
  const float e = ex2_approx(z * z * (-0.5f * kLog2e));
  float q = fmaf(t, 0.03567485511302948f, -0.15720340609550476f);
  q = fmaf(t, q, 0.206354022026062f);
  q = fmaf(t, q, -0.053684085607528687f);
  q = fmaf(t, q, 0.1285618394613266f);
  q = fmaf(t, q, 0.09991343319416046f);
  q = fmaf(t, q, 0.12075396627187729f);
  q = fmaf(t, q, 0.11962930113077164f);
  q = q * t * e;
  const float cdf = z > 0.f ? 1.f - q : q;
  value = z * cdf;
  if constexpr (SLOPE) slope = fmaf(z * 0.3989422804f, e, cdf);
}

template <bool SLOPE, int N>
__device__ __forceinline__ void gated_act(int act, const float (&z)[N], float (&value)[N],
                                          float (&slope)[N]) {
  switch (act) {
    case ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) act_silu<SLOPE>(z[i], value[i], slope[i]);
      break;
    case ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) act_gelu<SLOPE>(z[i], value[i], slope[i]);
      break;
    case ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) act_sigmoid<SLOPE>(z[i], value[i], slope[i]);
      break;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) act_tanh<SLOPE>(z[i], value[i], slope[i]);
  }
}

enum GgMode { GG_PROJ = 0, GG_DX = 1, GG_DW = 2 };

constexpr int kGgBM = 128;       // rows of a tile (TMEM lanes)
constexpr int kGgBK = 64;        // reduction depth of a stage: one 128-byte swizzle row of 16-bit
constexpr int kGgWindow = 4;     // stages between promotions of the fp32 variant (256 deep)
constexpr int kGgThreads = 320;
constexpr int kGgEpiWarps = 8;
constexpr int kGgGroup = 8;      // row tiles that share a pass over the column tiles (L2 reuse)

struct GgArgs {
  int64_t M, N;        // output rows and columns (GG_PROJ: of one projection; GG_DW: of one weight)
  int32_t tiles_m;     // over all halves
  int32_t tiles_n;
  int32_t half_tiles;  // GG_DW: row tiles of one weight; 0 = both weights' rows share a tile
  int32_t kblocks;     // stages of one segment
  int32_t segs;        // segments of the reduction
  int32_t splits;      // GG_DW: ranges of the reduction
  int32_t kb_per;      // stages per range
  uint32_t idesc;
  // epilogue
  void* out[2];        // GG_PROJ: out, or the dgate / dup planes; GG_DX: dx; GG_DW: dWg, dWu
  int64_t out_ld;
  int64_t plane;       // elements between planes of dgate / dup
  float* partial;      // GG_DW with splits > 1: [split][2][M][N]
  const void* bg;
  const void* bu;
  const void* dout;
  float* col_sums;     // backward GG_PROJ: [4 tiles_m][2][N] column sums of dgate and dup, or null
  int64_t dout_ld;
  int32_t act;
  int32_t vec;         // 16-byte stores (and dout loads) are aligned
  int* err;
};

// 128-byte-swizzled shared-memory descriptor. K-major: rows of 128 bytes, 8-row atoms `sbo` = 1024
// bytes apart (lbo unused). MN-major: blocks of [64 reduction rows][64 outputs], 8-row groups 1024
// bytes apart (sbo), blocks of 64 outputs `lbo` bytes apart.
__device__ __forceinline__ uint64_t gg_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version for sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

// kind::f16 instruction descriptor: D f32, A and B of one 16-bit type.
__host__ __device__ constexpr uint32_t gg_idesc(bool bf16, bool a_mn, bool b_mn, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kGgBM >> 4) << 24);
}

__device__ __forceinline__ void gg_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void gg_tma(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                       uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
      : "memory");
}

// v = a + b + c exactly, each of 8 significant bits (round to nearest, so the parts shrink by 2^-8
// and 2^-16 and the dropped products stay below 2^-25). A value that rounds past bf16's range is cut
// instead; one that is not finite stays whole in the first part.
__device__ __forceinline__ float gg_bf16_part(float v) {
  const float r = __bfloat162float(__float2bfloat16_rn(v));
  return fabsf(r) <= 3.4e38f || v != v ? r : __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
}
__device__ __forceinline__ void gg_split3(float v, float& a, float& b, float& c) {
  a = gg_bf16_part(v);
  const float r = v - a;
  b = r == r ? gg_bf16_part(r) : 0.f;
  c = r == r ? r - b : 0.f;
}

template <int MODE, int NB, int PA, int PB>
struct GgShape {
  static constexpr int kABytes = kGgBM * kGgBK * 2;
  static constexpr int kBBytes = NB * kGgBK * 2;
  static constexpr int kStage = PA * kABytes + PB * kBBytes;
  static constexpr int kStages = 200 * 1024 / kStage < 8 ? 200 * 1024 / kStage : 8;
  static constexpr int kSmem = kStages * kStage + 1024;  // + alignment of the first stage
  static constexpr bool kWindowed = PB == 3;             // fp32 inputs
  static constexpr int kAcc = kWindowed ? 2 * NB : NB;   // TMEM columns of one accumulator buffer
  static_assert(2 * kAcc <= 512, "TMEM budget");
  static_assert(kStages >= 2, "shared-memory budget");
};

struct GgItem {
  int mt, nt, split, kb0, kb1;
};

__device__ __forceinline__ GgItem gg_item(const GgArgs& A, int64_t item) {
  GgItem I;
  const int64_t tiles = (int64_t)A.tiles_m * A.tiles_n;
  I.split = (int)(item / tiles);
  const int64_t t = item - I.split * tiles;
  const int64_t per = (int64_t)kGgGroup * A.tiles_n;
  const int g = (int)(t / per);
  const int in = (int)(t - g * per);
  const int rows = min(kGgGroup, A.tiles_m - g * kGgGroup);
  I.mt = g * kGgGroup + in % rows;
  I.nt = in / rows;
  I.kb0 = I.split * A.kb_per;
  I.kb1 = min(A.kblocks * A.segs, I.kb0 + A.kb_per);
  return I;
}

// Four fp32 columns of one row to the output's type.
template <typename T, int COLS>
__device__ __forceinline__ void gg_store(T* dst, const float (&v)[COLS], int64_t left, bool vec) {
  constexpr int V = 16 / sizeof(T);
  if (vec && left >= COLS) {
#pragma unroll
    for (int q = 0; q < COLS / V; ++q) {
      float w[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = v[q * V + i];
      store_vec<T, V>(dst + q * V, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < COLS; ++i)
      if (i < left) dst[i] = from_f<T>(v[i]);
  }
}

// Column sums of 16 columns over the warp's 32 rows: each step halves the columns a lane still
// carries (16 shuffles where a reduction per column takes 80). Lane l ends with column l / 2.
__device__ __forceinline__ float gg_col_sum(const float (&v)[16], int lane) {
  float a[8];
  const bool h4 = lane & 16, h3 = lane & 8, h2 = lane & 4, h1 = lane & 2;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    a[i] = (h4 ? v[i + 8] : v[i]) + __shfl_xor_sync(0xffffffffu, h4 ? v[i] : v[i + 8], 16);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = (h3 ? a[i + 4] : a[i]) + __shfl_xor_sync(0xffffffffu, h3 ? a[i] : a[i + 4], 8);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    a[i] = (h2 ? a[i + 2] : a[i]) + __shfl_xor_sync(0xffffffffu, h2 ? a[i] : a[i + 2], 4);
  a[0] = (h1 ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, h1 ? a[0] : a[1], 2);
  return a[0] + __shfl_xor_sync(0xffffffffu, a[0], 1);
}

// 16 raw elements of one dout row (zeros past the edges).
template <typename T>
struct GgRow {
  static constexpr int kVecs = sizeof(T);  // 16 columns are 2 or 4 16-byte vectors
  uint4 raw[kVecs];
  __device__ __forceinline__ void load(const GgArgs& A, int64_t m, int64_t n) {
    const T* src = (const T*)A.dout + m * A.dout_ld + n;
    const int64_t left = m < A.M ? A.N - n : 0;
    if (A.vec && left >= 16) {
#pragma unroll
      for (int q = 0; q < kVecs; ++q) raw[q] = reinterpret_cast<const uint4*>(src)[q];
    } else {
      T* e = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = i < left ? src[i] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    return to_f(reinterpret_cast<const T*>(raw)[i]);
  }
};

// Epilogue of 16 columns of one output row; `bias` holds the columns' gate biases, then `step` floats
// on their up biases. BACK: PD planes of dgate and dup, 16-bit type D, and their column sums.
template <typename T, typename D, int PD, bool BACK>
__device__ __forceinline__ void gg_proj_store(const GgArgs& A, int64_t m, int64_t n,
                                              const float* bias, int step, const GgRow<T>& dy,
                                              float* col_sums, int lane, float (&g)[16],
                                              float (&u)[16]) {
  const int64_t left = A.N - n;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias + i);
    const float4 c = *reinterpret_cast<const float4*>(bias + step + i);
    g[i] += b.x, g[i + 1] += b.y, g[i + 2] += b.z, g[i + 3] += b.w;
    u[i] += c.x, u[i + 1] += c.y, u[i + 2] += c.z, u[i + 3] += c.w;
  }
  float value[16], slope[16];
  gated_act<BACK>(A.act, g, value, slope);
  if constexpr (!BACK) {
    if (m >= A.M || left <= 0) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = value[i] * u[i];
    gg_store<T, 16>((T*)A.out[0] + m * A.out_ld + n, g, left, A.vec);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = dy.get(i);
      g[i] = d * u[i] * slope[i];
      u[i] = d * value[i];
    }
    if (col_sums && left > 0) {  // uniform over the warp
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float s = gg_col_sum(h == 0 ? g : u, lane);
        if ((lane & 1) == 0 && (lane >> 1) < left) col_sums[h * A.N + n + (lane >> 1)] = s;
      }
    }
    if (m >= A.M || left <= 0) return;
    // The planes' leading dimension is a multiple of 8 columns and their base is aligned, so the
    // stores are vectors; columns up to the leading dimension past N are never read.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float(&v)[16] = h == 0 ? g : u;
      D* dst = (D*)A.out[h] + m * A.out_ld + n;
#pragma unroll
      for (int p = 0; p < PD; ++p) {
        gg_store<D, 16>(dst + p * A.plane, v, left, true);
        if (p + 1 < PD) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float r = v[i] - to_f(from_f<D>(v[i]));
            v[i] = r == r && fabsf(r) < 3.0e38f ? r : 0.f;
          }
        }
      }
    }
  }
}

// Epilogue of 16 columns of a GG_DX or GG_DW tile.
template <typename T, int MODE>
__device__ __forceinline__ void gg_plain_store(const GgArgs& A, const GgItem& I, int lane_row,
                                               int64_t n, float (&v)[16]) {
  int half = 0;
  int64_t m;
  if constexpr (MODE == GG_DW) {
    if (A.half_tiles == 0) {
      half = lane_row >> 6;
      m = lane_row & 63;
    } else {
      half = I.mt >= A.half_tiles;
      m = (int64_t)(I.mt - half * A.half_tiles) * kGgBM + lane_row;
    }
  } else {
    m = (int64_t)I.mt * kGgBM + lane_row;
  }
  if (m >= A.M || n >= A.N) return;
  if (MODE == GG_DW && A.splits > 1) {
    float* dst = A.partial + (((int64_t)I.split * 2 + half) * A.M + m) * A.N + n;
    gg_store<float, 16>(dst, v, A.N - n, A.N % 4 == 0);
  } else if (A.out[half]) {
    gg_store<T, 16>((T*)A.out[half] + m * A.out_ld + n, v, A.N - n, A.vec);
  }
}

// T: the caller's element type; D: the operands' 16-bit type; PA, PB: planes of the two operands;
// PD: planes of dgate and dup that a backward GG_PROJ writes (their products take PA = PD).
template <int MODE, int NB, int PA, int PB, typename T, typename D, int PD, bool BACK>
__global__ void __launch_bounds__(kGgThreads, 1)
    gated_gemm_kernel(const __grid_constant__ CUtensorMap a0, const __grid_constant__ CUtensorMap a1,
                      const __grid_constant__ CUtensorMap b0, const __grid_constant__ CUtensorMap b1,
                      const __grid_constant__ GgArgs A) {
  using S = GgShape<MODE, NB, PA, PB>;
  constexpr int STAGES = S::kStages;
  constexpr bool WIN = S::kWindowed;
  constexpr int BN = MODE == GG_PROJ ? NB / 2 : NB;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) float bias_tile[kGgEpiWarps][MODE == GG_PROJ ? 2 * (BN / 2) : 4];
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kGgEpiWarps);
    }
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const int64_t items = (int64_t)A.tiles_m * A.tiles_n * A.splits;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const GgItem I = gg_item(A, item);
        const int n0 = I.nt * BN;
        for (int kb = I.kb0; kb < I.kb1; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES) ok = mbar_wait_bounded(&empty[s], ((it / STAGES) & 1) ^ 1);
          if (!ok) break;
          const int seg = kb >= A.kblocks;
          const int k0 = (kb - seg * A.kblocks) * kGgBK;
          const uint32_t sa = base + s * S::kStage, sb = sa + PA * S::kABytes;
          mbar_arrive_expect_tx(&full[s], S::kStage);
#pragma unroll
          for (int p = 0; p < PA; ++p) {
            const uint32_t dst = sa + p * S::kABytes;
            if constexpr (MODE == GG_DW) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int half = A.half_tiles == 0 ? q : I.mt >= A.half_tiles;
                const int m0 = A.half_tiles == 0
                                   ? 0
                                   : (I.mt - half * A.half_tiles) * kGgBM + q * 64;
                gg_tma(dst + q * 8192, half ? &a1 : &a0, m0, k0, p, &full[s]);
              }
            } else {
              gg_tma(dst, MODE == GG_DX && seg ? &a1 : &a0, k0, I.mt * kGgBM, p, &full[s]);
            }
          }
#pragma unroll
          for (int p = 0; p < PB; ++p) {
            const uint32_t dst = sb + p * S::kBBytes;
            if constexpr (MODE == GG_PROJ) {
              gg_tma(dst, &b0, k0, n0, p, &full[s]);
              gg_tma(dst + BN * 128, &b1, k0, n0, p, &full[s]);
            } else {
#pragma unroll
              for (int q = 0; q < NB / 64; ++q)
                gg_tma(dst + q * 8192, MODE == GG_DX && seg ? &b1 : &b0, n0 + q * 64, k0, p,
                       &full[s]);
            }
          }
        }
      }
      if (!ok) {
        atomicExch(A.err, DEV_WAIT_TIMEOUT);
        drain_ring<STAGES>(full, it);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t kAdvA = MODE == GG_DW ? 2048 >> 4 : 32 >> 4;
      constexpr uint32_t kAdvB = MODE == GG_PROJ ? 32 >> 4 : 2048 >> 4;
      int it = 0, buf_it = 0;
      for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const GgItem I = gg_item(A, item);
        for (int w0 = I.kb0; ok && w0 < I.kb1;) {
          const int w1 = WIN ? min(I.kb1, w0 + kGgWindow) : I.kb1;
          const int buf = buf_it & 1;
          if (buf_it >= 2) ok = mbar_wait_bounded(&acc_empty[buf], ((buf_it >> 1) & 1) ^ 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + buf * S::kAcc;
          for (int kb = w0; kb < w1; ++kb, ++it) {
            const int s = it % STAGES;
            ok = mbar_wait_bounded(&full[s], (it / STAGES) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t sa = base + s * S::kStage, sb = sa + PA * S::kABytes;
#pragma unroll
            for (int ks = 0; ks < kGgBK / 16; ++ks) {
              uint64_t da[PA], db[PB];
#pragma unroll
              for (int p = 0; p < PA; ++p)
                da[p] = gg_desc(sa + p * S::kABytes, MODE == GG_DW ? 8192 : 16, 1024) + ks * kAdvA;
#pragma unroll
              for (int p = 0; p < PB; ++p)
                db[p] = gg_desc(sb + p * S::kBBytes, MODE == GG_PROJ ? 16 : 8192, 1024) + ks * kAdvB;
              const uint32_t first = kb > w0 || ks > 0;
              if constexpr (WIN) {
                const uint32_t ds = d + NB;
                gg_mma(ds, da[2], db[0], A.idesc, first);
                gg_mma(ds, da[1], db[1], A.idesc, 1);
                gg_mma(ds, da[0], db[2], A.idesc, 1);
                gg_mma(ds, da[1], db[0], A.idesc, 1);
                gg_mma(ds, da[0], db[1], A.idesc, 1);
                gg_mma(d, da[0], db[0], A.idesc, first);
              } else {
#pragma unroll
                for (int p = PA - 1; p >= 0; --p)
                  gg_mma(d, da[p], db[0], A.idesc, p == PA - 1 ? first : 1);
              }
            }
            mma_commit(&empty[s]);
          }
          if (!ok) break;
          mma_commit(&acc_full[buf]);
          ++buf_it;
          w0 = w1;
        }
      }
      if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int lane_row = quad * 32 + lane;
    constexpr int HC = BN / 2;  // output columns of this warp
    int buf_it = 0;
    for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const GgItem I = gg_item(A, item);
      const int64_t m = (int64_t)I.mt * kGgBM + lane_row;
      const int64_t n = (int64_t)I.nt * BN + half * HC;
      float* bias = bias_tile[warp - 2];
      GgRow<T> dy, dy_next;
      float* col_sums = nullptr;
      if constexpr (MODE == GG_PROJ) {
        // The tile's biases and first dout columns come in while the MMAs still run.
        for (int q = lane; q < 2 * HC; q += 32) {
          const int64_t c = n + q % HC;
          const T* b = (const T*)(q < HC ? A.bg : A.bu);
          bias[q] = b && c < A.N ? to_f(b[c]) : 0.f;
        }
        __syncwarp();
        if constexpr (BACK) {
          dy_next.load(A, m, n);
          if (A.col_sums) col_sums = A.col_sums + ((int64_t)I.mt * 4 + quad) * 2 * A.N;
        }
      }
      if constexpr (!WIN) {
        const int buf = buf_it & 1;
        ok = mbar_wait_bounded(&acc_full[buf], (buf_it >> 1) & 1);
        if (ok) {
          tc_fence_after();
          const uint32_t t = tmem + buf * S::kAcc + ((uint32_t)quad << 21) + half * HC;
#pragma unroll 1
          for (int c = 0; c < HC; c += 16) {
            if constexpr (MODE == GG_PROJ) {
              uint32_t rg[16], ru[16];
              tmem_ld16_async(t + c, rg);
              tmem_ld16_async(t + BN + c, ru);
              if constexpr (BACK) {
                dy = dy_next;
                if (c + 16 < HC) dy_next.load(A, m, n + c + 16);
              }
              tmem_wait_ld();
              float g[16], u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                g[i] = __uint_as_float(rg[i]);
                u[i] = __uint_as_float(ru[i]);
              }
              gg_proj_store<T, D, PD, BACK>(A, m, n + c, bias + c, HC, dy, col_sums, lane, g, u);
            } else {
              float v[16];
              tmem_ld16(t + c, v);
              gg_plain_store<T, MODE>(A, I, lane_row, n + c, v);
            }
          }
          tc_fence_before();
          __syncwarp();  // also: this tile's biases are read before the next tile's are written
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
          ++buf_it;
        }
      } else {
        // Windows: both accumulators are added to registers, the epilogue follows the last.
        constexpr int R = MODE == GG_PROJ ? 2 : 1;
        float acc[R][HC];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < HC; ++i) acc[r][i] = 0.f;
        for (int w0 = I.kb0; ok && w0 < I.kb1; w0 += kGgWindow) {
          const int buf = buf_it & 1;
          ok = mbar_wait_bounded(&acc_full[buf], (buf_it >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t t = tmem + buf * S::kAcc + ((uint32_t)quad << 21) + half * HC;
#pragma unroll
          for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int c = 0; c < HC; c += 16) {
              uint32_t big[16], small[16];
              tmem_ld16_async(t + r * BN + c, big);
              tmem_ld16_async(t + NB + r * BN + c, small);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                acc[r][c + i] += __uint_as_float(big[i]) + __uint_as_float(small[i]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
          ++buf_it;
        }
        if (ok) {
#pragma unroll
          for (int c = 0; c < HC; c += 16) {
            float v[R][16];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int i = 0; i < 16; ++i) v[r][i] = acc[r][c + i];
            if constexpr (MODE == GG_PROJ) {
              if constexpr (BACK) {
                dy = dy_next;
                if (c + 16 < HC) dy_next.load(A, m, n + c + 16);
              }
              gg_proj_store<T, D, PD, BACK>(A, m, n + c, bias + c, HC, dy, col_sums, lane, v[0],
                                            v[R - 1]);
            } else {
              gg_plain_store<T, MODE>(A, I, lane_row, n + c, v[0]);
            }
          }
          __syncwarp();
        }
      }
    }
    if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace gpb
