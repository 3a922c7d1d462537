// Shared by the feature-map operators (layer norm, gated unit, dropout): element types, 16-byte
// vectors, the device guard of their entry points and their argument checks. These operators take
// no provider: every call names its device and stream and brings its own workspace, so calls on
// different streams (or in captured graphs) share nothing that the caller did not pass twice.
#pragma once

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gpb_common.cuh"

namespace gpb {

// B200 has 148 SMs; grids and workspace sizes that depend on the count use the constant, so that a
// workspace query needs no device.
constexpr int kFeatSMs = 148;

// Makes `device` current for the scope and restores the caller's device afterwards: these calls
// are made from programs that own the current device themselves.
struct DeviceScope {
  int saved = -1;
  cudaError_t status;
  explicit DeviceScope(int device) {
    status = cudaGetDevice(&saved);
    if (status == cudaSuccess && saved != device)
      status = cudaSetDevice(device);
    else if (status == cudaSuccess)
      saved = -1;
  }
  ~DeviceScope() {
    if (saved >= 0) cudaSetDevice(saved);
  }
};

#define GPB_DEVICE_SCOPE(device)                                                              \
  ::gpb::DeviceScope gpb_scope_(device);                                                      \
  GPB_REQUIRE(gpb_scope_.status == cudaSuccess, GPB_ERR_CUDA, "device %d: %s", (int)(device), \
              cudaGetErrorString(gpb_scope_.status))

inline bool dtype_ok(int32_t dt) {
  return dt == GPB_DTYPE_F32 || dt == GPB_DTYPE_F16 || dt == GPB_DTYPE_BF16;
}
inline int dtype_bytes(int32_t dt) { return dt == GPB_DTYPE_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

inline bool overlaps(const void* a, int64_t abytes, const void* b, int64_t bbytes) {
  if (!a || !b || abytes <= 0 || bbytes <= 0) return false;
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)bbytes && y < x + (uintptr_t)abytes;
}

// Memory of a [rows][cols] block of leading dimension ld, or of a vector, in bytes.
struct Extent {
  const void* p;
  int64_t rows, width, stride;
};
inline Extent block_extent(const void* p, int64_t rows, int64_t cols, int64_t ld, int esize) {
  return {p, rows, cols * esize, ld * esize};
}
inline Extent flat_extent(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }
// Two blocks with one row stride may lie side by side (column ranges of one matrix): then no row of one
// reaches the columns of the other.
inline bool overlaps(const Extent& a, const Extent& b) {
  auto span = [](const Extent& e) {
    return e.rows > 0 && e.width > 0 ? (e.rows - 1) * e.stride + e.width : 0;
  };
  if (!overlaps(a.p, span(a), b.p, span(b))) return false;
  const int64_t stride = a.rows > 1 ? a.stride : b.stride;
  if (b.rows > 1 && b.stride != stride) return true;
  int64_t right = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p) % stride;  // of b's rows from a's
  if (right < 0) right += stride;
  return right < a.width || right + b.width > stride;
}
// Natural alignment of the element type (a view of a byte buffer may miss it).
inline bool elem_aligned(const void* p, int esize) { return ((uintptr_t)p % (uintptr_t)esize) == 0; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// VEC elements moved together: accesses of at most 16 bytes (a float32 weight vector beside 8 16-bit
// elements is two of them), so 16-byte alignment is enough for every type.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[VEC]) {
  const Pack<T, VEC> q = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = to_f(q.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[VEC]) {
  Pack<T, VEC> q;
#pragma unroll
  for (int i = 0; i < VEC; ++i) q.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = q;
}

// The VEC elements of 16 raw bytes as fp32 pairs, and back (rounded to nearest).
__device__ __forceinline__ void unpack16(const uint4& q, float2 (&o)[2], const float*) {
  o[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
  o[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
}
__device__ __forceinline__ void unpack16(const uint4& q, float2 (&o)[4], const __nv_bfloat16*) {
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
}
__device__ __forceinline__ void unpack16(const uint4& q, float2 (&o)[4], const __half*) {
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[2], const float*) {
  return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                    __float_as_uint(v[1].y));
}
template <typename H2>
__device__ __forceinline__ uint32_t bits32(const H2& h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[4], const __nv_bfloat16*) {
  return make_uint4(bits32(__float22bfloat162_rn(v[0])), bits32(__float22bfloat162_rn(v[1])),
                    bits32(__float22bfloat162_rn(v[2])), bits32(__float22bfloat162_rn(v[3])));
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[4], const __half*) {
  return make_uint4(bits32(__float22half2_rn(v[0])), bits32(__float22half2_rn(v[1])),
                    bits32(__float22half2_rn(v[2])), bits32(__float22half2_rn(v[3])));
}

// Column sums of `rows` partial rows [2][cols] to two vectors (either may be null): columns
// [32 chunk, 32 chunk + 32) by a block of 1024 threads, 32 along the rows of each, in a fixed order.
template <typename W>
__device__ __forceinline__ void column_join(const float* __restrict__ partial, int64_t rows,
                                            int64_t cols, W* a, W* b, int64_t chunk) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t c = chunk * 32 + lane;
  float s = 0.f;
  if (c < 2 * cols) {
#pragma unroll 8
    for (int64_t r = part; r < rows; r += 32) s += partial[r * 2 * cols + c];
  }
  sums[part][lane] = s;
  __syncthreads();
  s = sums[lane][part];  // transposed: warp `part` sums column `part`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t col = chunk * 32 + part;
  if (lane == 0 && col < 2 * cols) {
    W* dst = col < cols ? a : b;
    if (dst) dst[col < cols ? col : col - cols] = from_f<W>(s);
  }
}

// Opts a kernel into `bytes` of dynamic shared memory, once per kernel and device.
template <auto kernel>
int allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  GPB_CHECK_CUDA(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return GPB_OK;
  GPB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return GPB_OK;
}

}  // namespace gpb
