// Element-type conversion of a row-major block (a feature map computed in 16 bits hands float32
// inputs to the GP, and takes float32 gradients back). Rounds to nearest; HBM bound.
#include "features.cuh"

namespace gpb {

template <typename S, typename D>
__global__ void __launch_bounds__(256) cast_kernel(const S* __restrict__ x, int64_t x_ld,
                                                   D* __restrict__ out, int64_t out_ld,
                                                   int64_t rows, int64_t cols) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= rows * cols) return;
  const int64_t r = e / cols, c = e - r * cols;
  out[r * out_ld + c] = from_f<D>(to_f(x[r * x_ld + c]));
}

template <typename S>
static void cast_launch(int32_t dst, const void* x, int64_t x_ld, void* out, int64_t out_ld,
                        int64_t rows, int64_t cols, cudaStream_t st) {
  const unsigned grid = (unsigned)ceil_div(rows * cols, 256);
  switch (dst) {
    case GPB_DTYPE_F32:
      cast_kernel<S, float><<<grid, 256, 0, st>>>((const S*)x, x_ld, (float*)out, out_ld, rows, cols);
      break;
    case GPB_DTYPE_F16:
      cast_kernel<S, __half><<<grid, 256, 0, st>>>((const S*)x, x_ld, (__half*)out, out_ld, rows, cols);
      break;
    default:
      cast_kernel<S, __nv_bfloat16>
          <<<grid, 256, 0, st>>>((const S*)x, x_ld, (__nv_bfloat16*)out, out_ld, rows, cols);
  }
}

}  // namespace gpb

using namespace gpb;

extern "C" int gpb_cast(int32_t device, void* stream, int32_t out_dtype, int32_t x_dtype,
                        int64_t rows, int64_t cols, void* out_dev, int64_t out_ld,
                        const void* x_dev, int64_t x_ld) {
  clear_error();
  GPB_REQUIRE(dtype_ok(out_dtype) && dtype_ok(x_dtype), GPB_ERR_INVALID, "unknown element type");
  GPB_REQUIRE(rows >= 0 && cols >= 0, GPB_ERR_INVALID, "negative size");
  if (rows == 0 || cols == 0) return GPB_OK;
  GPB_REQUIRE(cols <= ((int64_t)1 << 38) / rows, GPB_ERR_INVALID, "%lld x %lld elements are too many",
              (long long)rows, (long long)cols);
  GPB_REQUIRE(out_dev && x_dev, GPB_ERR_INVALID, "null argument");
  GPB_REQUIRE(out_ld >= cols && x_ld >= cols, GPB_ERR_INVALID,
              "leading dimension below the %lld columns", (long long)cols);
  const int os = dtype_bytes(out_dtype), xs = dtype_bytes(x_dtype);
  GPB_REQUIRE(elem_aligned(out_dev, os) && elem_aligned(x_dev, xs), GPB_ERR_INVALID,
              "pointer is not aligned to its element type");
  GPB_REQUIRE(!overlaps(block_extent(out_dev, rows, cols, out_ld, os),
                        block_extent(x_dev, rows, cols, x_ld, xs)),
              GPB_ERR_INVALID, "out overlaps x");
  GPB_DEVICE_SCOPE(device);
  cudaStream_t st = (cudaStream_t)stream;
  switch (x_dtype) {
    case GPB_DTYPE_F32: cast_launch<float>(out_dtype, x_dev, x_ld, out_dev, out_ld, rows, cols, st); break;
    case GPB_DTYPE_F16: cast_launch<__half>(out_dtype, x_dev, x_ld, out_dev, out_ld, rows, cols, st); break;
    default: cast_launch<__nv_bfloat16>(out_dtype, x_dev, x_ld, out_dev, out_ld, rows, cols, st);
  }
  GPB_CHECK_CUDA(cudaGetLastError());
  return GPB_OK;
}
