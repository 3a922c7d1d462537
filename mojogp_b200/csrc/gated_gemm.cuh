// The gated unit's matrix products on the 5th-generation tensor cores (tcgen05, kind::f16).
//
// One persistent kernel, three products over 16-bit operands with fp32 accumulators in TMEM:
//   GG_PROJ  gate | up = x [Wg' | Wu']   tile 128 rows x (BN gate + BN up columns): both projections
//            of the same outputs share the x tile and one MMA, and the epilogue applies the
//            activation and the product (or, for the backward pass, forms dgate and dup);
//   GG_DX    dx = dgate Wg + dup Wu      one accumulation over two segments;
//   GG_DW    dWg = dgate' x, dWu = dup' x   the reduction runs over rows.
// A product with too few tiles for the SMs, or a 16-bit one with a longer reduction than an accumulator that
// truncates should take, splits its reduction over CTAs (fp32 partial sums, joined in split order; GG_PROJ's
// epilogue then runs in the join).
// x and the weights are read where they lie. A product whose reduction index is not the contiguous
// one takes its operand MN-major: the tensor core transposes, nothing is copied.
//
// fp32 inputs are exact sums of three bf16 planes (8 significant bits each; the weights are packed
// before the call; x comes in as fp32 tiles that four warps split into the planes the MMAs read, 4
// bytes an element from HBM instead of a pass of 10 and 6 per use), and
// a product keeps the six plane pairs above 2^-24 of it: hi hi apart from the five small ones, which
// have their own accumulator. The tensor core truncates where it adds, about 2^-26 of the accumulator
// per term, so after every kGgWindow blocks of the reduction the epilogue warps add both accumulators
// to registers in fp32 and the MMAs start again from zero.
//
// Wide 16-bit products run on CTA pairs (cta_group::2): one MMA covers 256 rows x 256 columns, each
// CTA holds its 128 rows of A and half of B's rows, so a stage is 32 KB per CTA where a CTA alone loads
// 48 KB for the same MMA time: alone, the tile stream ran at 73 bytes per clock and SM, which is what
// the L2 gives, with the tensor pipe 76 % busy. The pair's even CTA issues the MMAs; both CTAs' loads
// complete on its barriers, and its commits arrive at both. Forward bf16 8192 x 2048 -> 8192 386 us alone,
// 311 us in pairs (1.77 PFLOP/s, what a plain matrix product reaches: MMA and power bound); backward
// 8192 x 1024 -> 4096 304 us, of which the projections 119 (1.15 PFLOP/s: two outputs and a gradient
// pass through their epilogue), dx 87 (1.58) and the weight gradients 93 (1.48).
//
// 10 warps: TMA producer, MMA issuer, 8 epilogue warps (TMEM lane quadrant = warp % 4, two warps
// share a quadrant's columns). Tiles move by cp.async.bulk.tensor into 128-byte-swizzled stages;
// accumulators are double-buffered so that a tile's epilogue runs under the next tile's MMAs. Every
// wait is bounded: one that runs out sets the module's error word and ends the role.
#pragma once

#include <cuda.h>

#include <type_traits>

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
// (bf16, with single-CTA tiles: the backward projections at 8192 x 1024 -> 4096 315 us, 162 us with
// these; the forward pass at 8192 x 2048 -> 8192 467 and 402 us).
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
constexpr int kGgSplitBK = 32;   // the same where x is split: more and smaller stages in flight
constexpr int kGgWindow = 256;   // depth between promotions of the fp32 variant
constexpr int kGgEpiWarps = 8;
constexpr int kGgSplitWarps = 4;
constexpr int kGgRaw = 3;        // fp32 tiles in flight (a fourth's memory is the rows' transpose)
constexpr int kGgGroup = 8;      // row tiles that share a pass over the column tiles (L2 reuse)

struct GgArgs {
  int64_t M, N;        // output rows and columns (GG_PROJ: of one projection; GG_DW: of one weight)
  int32_t tiles_m;     // row tiles over all halves (pairs of them for CTA pairs)
  int32_t tiles_n;
  int32_t half_tiles;  // GG_DW: row tiles of one weight; 0 = both weights' rows share a tile
  int32_t kblocks;     // stages of one segment
  int32_t segs;        // segments of the reduction
  int32_t splits;      // ranges of the reduction
  int32_t kb_per;      // stages per range
  int32_t a_rows;      // GG_PROJ, GG_DX: rows of an A tile that are loaded (the rest feeds unused rows)
  uint32_t idesc;
  // epilogue
  void* out[2];        // GG_PROJ: out, or the dgate / dup planes; GG_DX: dx; GG_DW: dWg, dWu
  int64_t out_ld;
  int64_t plane;       // elements between planes of dgate / dup
  float* partial;      // with splits > 1: [split][2, GG_DX 1][M][N rounded up to 16]
  const void* bg;
  const void* bu;
  const void* dout;
  float* col_sums;     // backward GG_PROJ: [4 tiles_m][2][N] column sums of dgate and dup, or null
  uint32_t* largest;   // float16 backward: bits of the largest |dgate|, |dup| (gg_factor_exp)
  int32_t redo;        // float16 backward GG_PROJ: the pass that writes scaled factors
  int64_t dout_ld;
  int32_t act;
  int32_t vec;         // output rows (backward GG_PROJ: dout rows) are 2: 32-byte, 1: 16-byte aligned
  int* err;
};

// Shared-memory descriptor. K-major: rows of 2 BK bytes, swizzled over their length (128 or 64 bytes),
// 8-row atoms `sbo` apart (lbo unused). MN-major: 128-byte swizzled blocks of [BK reduction rows][64
// outputs], 8-row groups 1024 bytes apart (sbo), blocks of 64 outputs `lbo` bytes apart.
template <bool MN, int BK>
__device__ __forceinline__ uint64_t gg_desc(uint32_t addr) {
  constexpr uint32_t lbo = MN ? BK * 128 : 16, sbo = MN ? 1024 : 8 * 2 * BK;
  constexpr uint64_t swizzle = MN || BK == 64 ? 2 : 4;
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version for sm_100
  d |= swizzle << 61;
  return d;
}

// kind::f16 instruction descriptor: D f32, A and B of one 16-bit type.
__host__ __device__ constexpr uint32_t gg_idesc(bool bf16, bool a_mn, bool b_mn, int n,
                                                int m = kGgBM) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// One lane of a converged warp. A tcgen05.mma under `elect.sync` takes its descriptors from uniform
// registers; under `lane == 0` the compiler cannot know that one thread runs it.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
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

// The pair's forms.
__device__ __forceinline__ void gg_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void gg_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], "
      "%1;" ::"r"(smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void gg_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void gg_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// The same shared-memory object in the pair's even CTA.
__device__ __forceinline__ uint32_t gg_leader_addr(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
  return a;
}
// The even CTA's barrier learns that TMEM was read; nothing in memory is handed over (a cluster-wide
// release would wait for the epilogue's stores).
__device__ __forceinline__ void gg_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t gg_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void gg_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// A load of a pair: into this CTA's memory, completing on a barrier of the even CTA.
__device__ __forceinline__ void gg_tma_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
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

// The next bf16 part of a pair of fp32 values, which keep their remainders: three parts are the exact
// value (round to nearest, so they shrink by 2^-8 and 2^-16 and the dropped products stay below
// 2^-25). A value beyond bf16's largest (3.3895e38) or not finite leaves a NaN remainder, and makes
// what depends on it NaN; looking for one per pair cost a branch that halted the splitting warps
// (a stage took 6 us where its MMAs take 0.8).
template <typename D>
__device__ __forceinline__ uint32_t gg_part(float2& x) {
  uint32_t h;
  float2 f;
  if constexpr (std::is_same<D, __nv_bfloat16>::value) {
    h = bits32(__float22bfloat162_rn(x));
    f = make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xFFFF0000u));
  } else {
    const __half2 v = __float22half2_rn(x);
    h = bits32(v);
    f = __half22float2(v);
  }
  x = __ffma2_rn(f, make_float2(-1.f, -1.f), x);
  return h;
}

// fp32 x is GG_PROJ's A operand and GG_DW's B operand.
__host__ __device__ constexpr bool gg_splits(int mode, int pb) { return pb == 3 && mode != GG_DX; }

template <int MODE, int NB, int PA, int PB, int CTAS>
struct GgShape {
  static constexpr bool kSplit = gg_splits(MODE, PB);
  static_assert(CTAS == 1 || (PA == 1 && PB == 1 && NB == 256), "pairs: wide 16-bit products");
  static constexpr int kBK = kSplit ? kGgSplitBK : kGgBK;
  static constexpr int kThreads = 32 * (2 + kGgEpiWarps + (kSplit ? kGgSplitWarps : 0));
  static constexpr int kABytes = kGgBM * kBK * 2;
  static constexpr int kBBytes = NB / CTAS * kBK * 2;
  static constexpr int kStage = PA * kABytes + PB * kBBytes;
  // The part of a stage that TMA writes; the splitting warps write the rest, from a ring of fp32 tiles.
  static constexpr bool kTmaA = !(kSplit && MODE == GG_PROJ), kTmaB = !(kSplit && MODE == GG_DW);
  static constexpr int kTmaBytes = (kTmaA ? PA * kABytes : 0) + (kTmaB ? PB * kBBytes : 0);
  static constexpr int kPlane = kTmaA ? kBBytes : kABytes;  // of the split operand
  static constexpr int kRaw = kSplit ? 2 * kPlane : 0;
  static constexpr int kRest = kGgRaw * kRaw;
  static constexpr int kStages =
      (200 * 1024 - kRest) / kStage < 8 ? (200 * 1024 - kRest) / kStage : 8;
  static constexpr int kSmem = kStages * kStage + kRest + 1024;  // + alignment of the first stage
  static constexpr bool kWindowed = PB == 3;             // fp32 inputs
  static constexpr int kWindow = kGgWindow / kBK;        // stages between promotions
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

// A whole 32-byte sector in one access (16-byte stores of a thread's own row leave half-written
// sectors to the L2).
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x),
               "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// Unaligned rows go through a warp's own 32 x 16 tile of shared memory, so that 16 lanes share a row:
// a lane's own row, element by element, makes every access 32 sectors of one element each.
constexpr int kGgTileLd = 17;  // words per row of the tile
constexpr int kGgTile = 32 * kGgTileLd;

// 16 columns of the warp's 32 rows, of which lane holds its own row; rows start at `row0` (lane 0's).
template <typename T>
__device__ __forceinline__ void gg_store_rows(T* out, int64_t ld, int64_t row0, int64_t rows, int64_t n,
                                              const float (&v)[16], int64_t left, float* tile,
                                              int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[lane * kGgTileLd + i] = v[i];
  __syncwarp();
  const int c = lane & 15;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 2 * i + (lane >> 4);
    if (row0 + r < rows && c < left) out[(row0 + r) * ld + n + c] = from_f<T>(tile[r * kGgTileLd + c]);
  }
  __syncwarp();
}

// float16 dgate and dup are written as they are, and their largest magnitude is found on the way. If that
// is 2^15 or more, where float16 ends, or below 2^-4, where the half of its smallest step (2^-25) is more
// than 2^-21 of it, a second pass writes them times 2^k, the largest one then in [2^13, 2^14); GG_DX and GG_DW
// divide by it again. The second pass ends at once where k is 0. (A maximum is the same in any order, so
// results repeat.) Unscaled, a finite factor beyond 65504 made a row of dx and a column of dW NaN, and a
// small gradient vanished. Backward 8192 x 1024 -> 4096: bf16, which needs none of this, 329 us, fp16 348, and
// 482 where it scales; 16 x 2048 -> 8192 75, 82 and 95. k, from the largest magnitude's bits; 0 where all factors are.
template <typename D>
constexpr bool kGgScaled = std::is_same<D, __half>::value;
__device__ __forceinline__ int gg_factor_exp(uint32_t bits) {
  if (bits == 0) return 0;
  const int e = (int)(bits >> 23) - 127;
  return e >= -4 && e < 15 ? 0 : min(13 - e, 126);
}
// A factor's part in the maximum: one that is not finite stays its own and has none.
__device__ __forceinline__ float gg_magnitude(float v) {
  return fabsf(v) < __int_as_float(0x7F800000) ? fabsf(v) : 0.f;
}
__device__ __forceinline__ float gg_pow2(int k) { return __int_as_float((k + 127) << 23); }

// 16 columns of the lane's row m to the output's type; vec: 2 = 32-byte aligned rows, 1 = 16-byte, 0 =
// neither. The whole warp takes part.
template <typename T>
__device__ __forceinline__ void gg_store(T* out, int64_t ld, int64_t m, int64_t rows, int64_t n,
                                         const float (&v)[16], int64_t left, int vec, float* tile,
                                         int lane) {
  constexpr int V = 16 / sizeof(T), Q = 16 / V;
  if (left <= 0) return;
  if (vec && left >= 16) {
    if (m >= rows) return;
    T* dst = out + m * ld + n;
    uint4 raw[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float2 w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = make_float2(v[q * V + 2 * i], v[q * V + 2 * i + 1]);
      raw[q] = pack16(w, (const T*)nullptr);
    }
#pragma unroll
    for (int q = 0; q < Q; q += 2) {
      if (vec == 2) {
        store32(dst + q * V, raw[q], raw[q + 1]);
      } else {
        reinterpret_cast<uint4*>(dst)[q] = raw[q];
        reinterpret_cast<uint4*>(dst)[q + 1] = raw[q + 1];
      }
    }
  } else {
    gg_store_rows<T>(out, ld, m - lane, rows, n, v, left, tile, lane);
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
  __device__ __forceinline__ void load(const GgArgs& A, int64_t m, int64_t n, float* tile, int lane) {
    const T* src = (const T*)A.dout + m * A.dout_ld + n;
    const int64_t left = A.N - n;
    if (A.splits > 1) return;  // the join reads dout
    if (A.vec && left >= 16) {
#pragma unroll
      for (int q = 0; q < kVecs; ++q)
        raw[q] = m < A.M ? reinterpret_cast<const uint4*>(src)[q] : make_uint4(0, 0, 0, 0);
    } else {
      const int c = lane & 15;
      const int64_t row0 = m - lane;
      T* t = reinterpret_cast<T*>(tile);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4);
        t[r * kGgTileLd + c] = row0 + r < A.M && c < left
                                   ? ((const T*)A.dout)[(row0 + r) * A.dout_ld + n + c]
                                   : from_f<T>(0.f);
      }
      __syncwarp();
      T* e = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = t[lane * kGgTileLd + i];
      __syncwarp();
    }
  }
  __device__ __forceinline__ float get(int i) const {
    return to_f(reinterpret_cast<const T*>(raw)[i]);
  }
};

// 16 fp32 partial sums of a row: whole sectors (rows are padded to a multiple of 16 columns).
__device__ __forceinline__ void gg_store_partial(float* dst, const float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 16; q += 8)
    store32(dst + q,
            make_uint4(__float_as_uint(v[q]), __float_as_uint(v[q + 1]), __float_as_uint(v[q + 2]),
                       __float_as_uint(v[q + 3])),
            make_uint4(__float_as_uint(v[q + 4]), __float_as_uint(v[q + 5]),
                       __float_as_uint(v[q + 6]), __float_as_uint(v[q + 7])));
}

// Epilogue of 16 columns of one output row; `bias` holds the columns' gate biases, then `step` floats
// on their up biases. BACK: PD planes of dgate and dup, 16-bit type D, and their column sums.
template <typename T, typename D, int PD, bool BACK>
__device__ __forceinline__ void gg_proj_store(const GgArgs& A, int split, int64_t m, int64_t n,
                                              const float* bias, int step, const GgRow<T>& dy,
                                              float* col_sums, float* tile, int lane, float (&g)[16],
                                              float (&u)[16], float scale, float& largest) {
  const int64_t left = A.N - n;
  if (A.splits > 1) {
    const int64_t ld = (A.N + 15) / 16 * 16;
    if (m < A.M && left > 0) {
      gg_store_partial(A.partial + ((int64_t)split * 2 * A.M + m) * ld + n, g);
      gg_store_partial(A.partial + (((int64_t)split * 2 + 1) * A.M + m) * ld + n, u);
    }
    return;
  }
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
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = value[i] * u[i];
    gg_store<T>((T*)A.out[0], A.out_ld, m, A.M, n, g, left, A.vec, tile, lane);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = dy.get(i);
      g[i] = d * u[i] * slope[i];
      u[i] = d * value[i];
    }
    if (m >= A.M) {
      // Past the last row x and dout are zeros, but a weight or bias that is not finite is not.
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] = u[i] = 0.f;
    }
    if constexpr (kGgScaled<D>) {
#pragma unroll
      for (int i = 0; i < 16; ++i) largest = fmaxf(largest, fmaxf(gg_magnitude(g[i]), gg_magnitude(u[i])));
    }
    if (col_sums && left > 0) {  // uniform over the warp
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float s = gg_col_sum(h == 0 ? g : u, lane);
        if ((lane & 1) == 0 && (lane >> 1) < left) col_sums[h * A.N + n + (lane >> 1)] = s;
      }
    }
    if (m >= A.M || left <= 0) return;
    // The planes' leading dimension is a multiple of 16 columns and their base is aligned, so the
    // stores are whole sectors; columns up to the leading dimension past N are never read.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float(&v)[16] = h == 0 ? g : u;
      D* dst = (D*)A.out[h] + m * A.out_ld + n;
      float2 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = make_float2(v[2 * i], v[2 * i + 1]);
        if constexpr (kGgScaled<D>) x[i] = __fmul2_rn(x[i], make_float2(scale, scale));
      }
#pragma unroll
      for (int p = 0; p < PD; ++p) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = gg_part<D>(x[i]);
        store32(dst + p * A.plane, make_uint4(w[0], w[1], w[2], w[3]),
                make_uint4(w[4], w[5], w[6], w[7]));
      }
    }
  }
}

// Epilogue of 16 columns of a GG_DX or GG_DW tile. The warp's 32 rows belong to one weight (halves of a
// shared tile are 64 rows).
template <typename T, typename D, int MODE>
__device__ __forceinline__ void gg_plain_store(const GgArgs& A, int split, int mt, int lane_row,
                                               int64_t n, float (&v)[16], float* tile, int lane,
                                               float scale) {
  if constexpr (kGgScaled<D>) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= scale;
  }
  int half = 0;
  int64_t m;
  if constexpr (MODE == GG_DW) {
    if (A.half_tiles == 0) {
      half = lane_row >> 6;
      m = lane_row & 63;
    } else {
      half = mt >= A.half_tiles;
      m = (int64_t)(mt - half * A.half_tiles) * kGgBM + lane_row;
    }
  } else {
    m = (int64_t)mt * kGgBM + lane_row;
  }
  const int64_t left = A.N - n;
  if (A.splits > 1) {
    constexpr int HALVES = MODE == GG_DW ? 2 : 1;
    const int64_t ld = (A.N + 15) / 16 * 16;
    if (m < A.M && left > 0)
      gg_store_partial(A.partial + (((int64_t)split * HALVES + half) * A.M + m) * ld + n, v);
  } else if (A.out[half]) {
    gg_store<T>((T*)A.out[half], A.out_ld, m, A.M, n, v, left, A.vec, tile, lane);
  }
}

// Splits an fp32 tile into planes: 128 threads, each UNITS runs of 8 elements, 128 runs apart. ROW
// elements to a row of the tile; planes' rows are swizzled as TMA writes them.
template <int UNITS, int ROW>
__device__ __forceinline__ void gg_split_tile(int tid, uint32_t raw, uint32_t tile, uint32_t plane) {
  float2 v[UNITS][4];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const uint32_t at = raw + (u * 128 + tid) * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[u][2 * h].x), "=f"(v[u][2 * h].y), "=f"(v[u][2 * h + 1].x),
                     "=f"(v[u][2 * h + 1].y)
                   : "r"(at + 16 * h));
  }
  constexpr int RUNS = ROW / 8;
  const int r0 = tid / RUNS, c0 = tid % RUNS;  // 128 runs on: the same swizzle
  const int c = ROW == 64 ? c0 ^ (r0 & 7) : c0 ^ ((r0 >> 1) & 3);
  const uint32_t at0 = tile + r0 * (ROW * 2) + c * 16;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = gg_part<__nv_bfloat16>(v[u][i]);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at0 + u * 2048 + k * plane),
                   "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3])
                   : "memory");
    }
  }
}

// T: the caller's element type; D: the operands' 16-bit type; PA, PB: planes of the two operands;
// PD: planes of dgate and dup that a backward GG_PROJ writes (their products take PA = PD).
template <int MODE, int NB, int PA, int PB, typename T, typename D, int PD, bool BACK, int CTAS>
__global__ void __cluster_dims__(CTAS, 1, 1)
    __launch_bounds__((GgShape<MODE, NB, PA, PB, CTAS>::kThreads), 1)
    gated_gemm_kernel(const __grid_constant__ CUtensorMap a0, const __grid_constant__ CUtensorMap a1,
                      const __grid_constant__ CUtensorMap b0, const __grid_constant__ CUtensorMap b1,
                      const __grid_constant__ GgArgs A) {
  using S = GgShape<MODE, NB, PA, PB, CTAS>;
  constexpr bool PAIR = CTAS == 2;
  constexpr int STAGES = S::kStages;
  constexpr bool WIN = S::kWindowed;
  constexpr int BN = MODE == GG_PROJ ? NB / 2 : NB;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  __shared__ __align__(8) uint64_t raw_full[kGgRaw], raw_empty[kGgRaw];
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) float bias_tile[kGgEpiWarps][MODE == GG_PROJ ? 2 * (BN / 2) : 4];
  __shared__ float row_tile[kGgEpiWarps][kGgTile];
  float scale = 1.f, largest = 0.f;  // of float16 factors
  if constexpr (kGgScaled<D> && (BACK || MODE != GG_PROJ)) {
    if (MODE != GG_PROJ || A.redo) {
      const int k = gg_factor_exp(*A.largest);
      if (MODE == GG_PROJ && k == 0) return;  // the whole grid
      scale = gg_pow2(MODE == GG_PROJ ? k : -k);
    }
  }
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t raw = base + STAGES * S::kStage;
  constexpr int BK = S::kBK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1 + (S::kSplit ? kGgSplitWarps : 0));
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], CTAS * kGgEpiWarps);
    }
    for (int s = 0; s < kGgRaw; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], kGgSplitWarps);
    }
    fence_barrier_init();
  }
  const int rank = PAIR ? (int)gg_cluster_rank() : 0;
  if (warp == 1) {
    if constexpr (PAIR)
      gg_alloc_pair(&tmem_base, 512);
    else
      tmem_alloc(&tmem_base, 512);
  }
  tc_fence_before();
  if constexpr (PAIR)
    gg_cluster_sync();  // the other CTA's barriers are initialised, too
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  // A pair works on one item: two row tiles of one column tile.
  const int64_t first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  const int64_t items = (int64_t)A.tiles_m * A.tiles_n * A.splits;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0, raw_it = 0;
      for (int64_t item = first; ok && item < items; item += step) {
        const GgItem I = gg_item(A, item);
        const int n0 = I.nt * BN;
        for (int kb = I.kb0; kb < I.kb1; ++kb, ++it) {
          const int s = it % STAGES;
          const int seg = kb >= A.kblocks;
          const int k0 = (kb - seg * A.kblocks) * BK;
          if constexpr (S::kSplit) {
            const int q = it % kGgRaw;
            if (it >= kGgRaw) ok = mbar_wait_bounded(&raw_empty[q], ((it / kGgRaw) & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&raw_full[q], MODE == GG_PROJ ? A.a_rows * (BK * 4) : S::kRaw);
            const uint32_t dst = raw + q * S::kRaw;
            if constexpr (MODE == GG_PROJ) {
              gg_tma(dst, &a0, k0, I.mt * kGgBM, 0, &raw_full[q]);
            } else {
#pragma unroll
              for (int c = 0; c < NB / 64; ++c)
                gg_tma(dst + c * BK * 64 * 4, &b0, n0 + c * 64, k0, 0, &raw_full[q]);
            }
            ++raw_it;
          }
          if (it >= STAGES) ok = mbar_wait_bounded(&empty[s], ((it / STAGES) & 1) ^ 1);
          if (!ok) break;
          const uint32_t sa = base + s * S::kStage, sb = sa + PA * S::kABytes;
          const int mt = I.mt * CTAS + rank;
          // Both CTAs' bytes are expected by the even one (the odd one's may come first).
          uint32_t pair_bar = 0;
          if constexpr (PAIR) pair_bar = gg_leader_addr(&full[s]);
          if (rank == 0) {
            int bytes = CTAS * S::kTmaBytes;
            if constexpr (CTAS == 1 && S::kTmaA && MODE != GG_DW)
              bytes -= PA * (kGgBM - A.a_rows) * (2 * BK);
            mbar_arrive_expect_tx(&full[s], bytes);
          }
          auto tma = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2) {
            if constexpr (PAIR)
              gg_tma_pair(dst, map, c0, c1, c2, pair_bar);
            else
              gg_tma(dst, map, c0, c1, c2, &full[s]);
          };
#pragma unroll
          for (int p = 0; p < (S::kTmaA ? PA : 0); ++p) {
            const uint32_t dst = sa + p * S::kABytes;
            if constexpr (MODE == GG_DW) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int half = A.half_tiles == 0 ? q : mt >= A.half_tiles;
                const int m0 =
                    A.half_tiles == 0 ? 0 : (mt - half * A.half_tiles) * kGgBM + q * 64;
                tma(dst + q * (BK * 128), half ? &a1 : &a0, m0, k0, p);
              }
            } else {
              tma(dst, MODE == GG_DX && seg ? &a1 : &a0, k0, mt * kGgBM, p);
            }
          }
#pragma unroll
          for (int p = 0; p < (S::kTmaB ? PB : 0); ++p) {
            const uint32_t dst = sb + p * S::kBBytes;
            if constexpr (MODE == GG_PROJ) {
              if constexpr (PAIR) {  // one projection's rows each
                tma(dst, rank ? &b1 : &b0, k0, n0, p);
              } else {
                tma(dst, &b0, k0, n0, p);
                tma(dst + BN * (2 * BK), &b1, k0, n0, p);
              }
            } else {
#pragma unroll
              for (int q = 0; q < NB / CTAS / 64; ++q)
                tma(dst + q * (BK * 128), MODE == GG_DX && seg ? &b1 : &b0,
                    n0 + (rank * (NB / CTAS) + q * 64), k0, p);
            }
          }
        }
      }
      if (!ok) {
        atomicExch(A.err, DEV_WAIT_TIMEOUT);
        if (rank == 0) drain_ring<STAGES>(full, it);  // a pair's loads complete on the even CTA
        if constexpr (S::kSplit) drain_ring<kGgRaw>(raw_full, raw_it);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp walks the stages and one elected lane issues: its waits must not part the warp.
      auto wait = [&](uint64_t* bar, int parity) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
        return ok;
      };
      constexpr uint32_t kAdvA = MODE == GG_DW ? 2048 >> 4 : 32 >> 4;
      constexpr uint32_t kAdvB = MODE == GG_PROJ ? 32 >> 4 : 2048 >> 4;
      int it = 0, buf_it = 0;
      for (int64_t item = first; ok && item < items; item += step) {
        const GgItem I = gg_item(A, item);
        for (int w0 = I.kb0; ok && w0 < I.kb1;) {
          const int w1 = WIN ? min(I.kb1, w0 + S::kWindow) : I.kb1;
          const int buf = buf_it & 1;
          if (buf_it >= 2 && !wait(&acc_empty[buf], ((buf_it >> 1) & 1) ^ 1)) break;
          const uint32_t d = tmem + buf * S::kAcc;
          for (int kb = w0; kb < w1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!wait(&full[s], (it / STAGES) & 1)) break;
            tc_fence_after();
            const uint32_t sa = base + s * S::kStage, sb = sa + PA * S::kABytes;
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks) {
                uint64_t da[PA], db[PB];
#pragma unroll
                for (int p = 0; p < PA; ++p)
                  da[p] = gg_desc<MODE == GG_DW, BK>(sa + p * S::kABytes) + ks * kAdvA;
#pragma unroll
                for (int p = 0; p < PB; ++p)
                  db[p] = gg_desc<MODE != GG_PROJ, BK>(sb + p * S::kBBytes) + ks * kAdvB;
                const uint32_t first_mma = kb > w0 || ks > 0;
                if constexpr (WIN) {
                  const uint32_t ds = d + NB;
                  gg_mma(ds, da[2], db[0], A.idesc, first_mma);
                  gg_mma(ds, da[1], db[1], A.idesc, 1);
                  gg_mma(ds, da[0], db[2], A.idesc, 1);
                  gg_mma(ds, da[1], db[0], A.idesc, 1);
                  gg_mma(ds, da[0], db[1], A.idesc, 1);
                  gg_mma(d, da[0], db[0], A.idesc, first_mma);
                } else {
#pragma unroll
                  for (int p = PA - 1; p >= 0; --p)
                    if constexpr (PAIR)
                      gg_mma_pair(d, da[p], db[0], A.idesc, first_mma);
                    else
                      gg_mma(d, da[p], db[0], A.idesc, p == PA - 1 ? first_mma : 1);
                }
              }
              if constexpr (PAIR) {
                gg_commit_pair(&empty[s]);
                if (kb + 1 == w1) gg_commit_pair(&acc_full[buf]);
              } else {
                mma_commit(&empty[s]);
                if (kb + 1 == w1) mma_commit(&acc_full[buf]);
              }
            }
            __syncwarp();
          }
          ++buf_it;
          w0 = w1;
        }
      }
      if (!ok && lane == 0) atomicExch(A.err, DEV_WAIT_TIMEOUT);
    }
  } else if (S::kSplit && warp >= 2 + kGgEpiWarps) {
    if constexpr (S::kSplit) {
      const int tid = threadIdx.x - 32 * (2 + kGgEpiWarps);
      int it = 0;
      for (int64_t item = first; ok && item < items; item += step) {
        const GgItem I = gg_item(A, item);
        for (int kb = I.kb0; kb < I.kb1; ++kb, ++it) {
          const int s = it % STAGES, q = it % kGgRaw;
          ok = mbar_wait_bounded(&raw_full[q], (it / kGgRaw) & 1);
          if (ok && it >= STAGES) ok = mbar_wait_bounded(&empty[s], ((it / STAGES) & 1) ^ 1);
          if (!ok) break;
          const uint32_t tile = base + s * S::kStage + (MODE == GG_PROJ ? 0 : PA * S::kABytes);
          gg_split_tile<S::kPlane / 2048, MODE == GG_PROJ ? BK : 64>(tid, raw + q * S::kRaw, tile,
                                                                     S::kPlane);
          fence_proxy_async_smem();
          __syncwarp();  // the warp's reads of the fp32 tile are done too
          if (lane == 0) {
            mbar_arrive(&raw_empty[q]);
            mbar_arrive(&full[s]);
          }
        }
      }
      if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int lane_row = quad * 32 + lane;
    constexpr int HC = BN / 2;  // output columns of this warp
    int buf_it = 0;
    for (int64_t item = first; ok && item < items; item += step) {
      const GgItem I = gg_item(A, item);
      const int mt = I.mt * CTAS + rank;
      const int64_t m = (int64_t)mt * kGgBM + lane_row;
      const int64_t n = (int64_t)I.nt * BN + half * HC;
      float* bias = bias_tile[warp - 2];
      float* tile = row_tile[warp - 2];
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
          dy_next.load(A, m, n, tile, lane);
          if (A.col_sums && (int64_t)mt * kGgBM < A.M) col_sums = A.col_sums + ((int64_t)mt * 4 + quad) * 2 * A.N;
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
            // The accumulator is free once its last columns are in registers, before they are worked on.
            auto release = [&]() {
              if (c + 16 < HC) return;
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if constexpr (PAIR)
                  gg_arrive_cluster(gg_leader_addr(&acc_empty[buf]));
                else
                  mbar_arrive(&acc_empty[buf]);
              }
            };
            if constexpr (MODE == GG_PROJ) {
              uint32_t rg[16], ru[16];
              tmem_ld16_async(t + c, rg);
              tmem_ld16_async(t + BN + c, ru);
              if constexpr (BACK) {
                dy = dy_next;
                if (c + 16 < HC) dy_next.load(A, m, n + c + 16, tile, lane);
              }
              tmem_wait_ld();
              release();
              float g[16], u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                g[i] = __uint_as_float(rg[i]);
                u[i] = __uint_as_float(ru[i]);
              }
              gg_proj_store<T, D, PD, BACK>(A, I.split, m, n + c, bias + c, HC, dy, col_sums, tile, lane, g, u,
                                            scale, largest);
            } else {
              float v[16];
              tmem_ld16(t + c, v);
              release();
              gg_plain_store<T, D, MODE>(A, I.split, mt, lane_row, n + c, v, tile, lane, scale);
            }
          }
          __syncwarp();  // this tile's biases are read before the next tile's are written
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
        for (int w0 = I.kb0; ok && w0 < I.kb1; w0 += S::kWindow) {
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
                if (c + 16 < HC) dy_next.load(A, m, n + c + 16, tile, lane);
              }
              gg_proj_store<T, D, PD, BACK>(A, I.split, m, n + c, bias + c, HC, dy, col_sums, tile, lane, v[0],
                                            v[R - 1], scale, largest);
            } else {
              gg_plain_store<T, D, MODE>(A, I.split, mt, lane_row, n + c, v[0], tile, lane, scale);
            }
          }
          __syncwarp();
        }
      }
    }
    if (!ok) atomicExch(A.err, DEV_WAIT_TIMEOUT);
    if constexpr (kGgScaled<D> && MODE == GG_PROJ && BACK) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
      if (lane == 0 && !A.redo && A.splits == 1 && top > 0) atomicMax(A.largest, top);
    }
  }
  tc_fence_before();
  if constexpr (PAIR)
    gg_cluster_sync();  // the even CTA's MMAs read the odd one's memory, and its barriers are used
  else
    __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      gg_dealloc_pair(tmem, 512);
    else
      tmem_dealloc(tmem, 512);
  }
}

}  // namespace gpb
