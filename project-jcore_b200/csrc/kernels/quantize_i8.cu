// 8-bit operands of nplk_gemm_i8: a scale for each row (token) or column
// (output channel) and the rounded quotients.
//
//   scale = max(max|x| / 127, 2^-126), q = rint(x / scale).
//
// The lower limit keeps the quotient finite where max|x| / 127 is denormal.
// The quotient is the correctly rounded fp32 one: q then depends on x alone,
// not on how a kernel forms it.
#include <math_constants.h>

#include "nplk_host.h"
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr int kThreads = 256;

// Largest magnitude so far, where a NaN stays (fmaxf would drop it): for
// non-negative floats and NaN without its sign the bit patterns are in order.
__device__ __forceinline__ uint32_t magnitude_bits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

__device__ __forceinline__ float scale_of(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  if (top_bits > 0x7f800000u) return CUDART_NAN_F;
  return fmaxf(top / 127.0f, 1.17549435e-38f);  // +infinity stays
}

__device__ __forceinline__ int8_t quantize(float v, float scale, bool finite) {
  return finite ? static_cast<int8_t>(__float2int_rn(v / scale)) : int8_t(0);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int w = 0; w < kThreads / 32; ++w) t = max(t, red[w]);
  return t;
}

// One block per line; element j of line i is x[i * line_step + j * step].
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_lines_kernel(int64_t length, const T *x, int64_t line_step, int64_t step, int8_t *q,
                          int64_t ldq, float *scale_out) {
  __shared__ uint32_t red[kThreads / 32];
  const int64_t line = blockIdx.x;
  const T *xl = x + line * line_step;
  uint32_t top = 0;
  for (int64_t j = threadIdx.x; j < length; j += kThreads)
    top = max(top, magnitude_bits(to_float(xl[j * step])));
  const float scale = scale_of(block_max(top, red));
  if (threadIdx.x == 0) scale_out[line] = scale;
  const bool finite = scale < CUDART_INF_F;
  for (int64_t j = threadIdx.x; j < length; j += kThreads)
    q[line * ldq + j] = quantize(to_float(xl[j * step]), scale, finite);
}

int quantize_lines(void *stream, int64_t rows, int64_t cols, int dtype, const void *x,
                   int64_t ldx, int8_t *q, int64_t ldq, float *scale, bool by_rows) {
  const int size = dtype_bytes(dtype);
  if (rows < 1 || cols < 1 || !size || !x || !q || !scale || ldx < cols ||
      ldq < (by_rows ? cols : rows))
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % size) return kErrInvalidArg;
  if (rows >= (int64_t(1) << 31) || cols >= (int64_t(1) << 31)) return kErrUnsupported;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(by_rows ? rows : cols);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    quantize_lines_kernel<T><<<grid, kThreads, 0, s>>>(by_rows ? cols : rows,
                                                       static_cast<const T *>(x),
                                                       by_rows ? ldx : 1, by_rows ? 1 : ldx, q,
                                                       ldq, scale);
  };
  if (dtype == NPLK_DTYPE_FP32) go(float{});
  else if (dtype == NPLK_DTYPE_FP16) go(__half{});
  else go(__nv_bfloat16{});
  count_launch();
  return launch_result();
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_quantize_rows(void *stream, int64_t rows, int64_t cols, int dtype,
                                  const void *x, int64_t ldx, int8_t *q, int64_t ldq,
                                  float *scale) {
  return quantize_lines(stream, rows, cols, dtype, x, ldx, q, ldq, scale, true);
}

extern "C" int nplk_quantize_cols(void *stream, int64_t rows, int64_t cols, int dtype,
                                  const void *x, int64_t ldx, int8_t *q, int64_t ldq,
                                  float *scale) {
  return quantize_lines(stream, rows, cols, dtype, x, ldx, q, ldq, scale, false);
}
