// Weights in 4 bits by groups along K: two to a byte, the even one in the low half;
// a weight is scale * (nibble - zero), zero 8 where none are stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "npl_kernels.h"
#include "typed_io.cuh"

namespace nplk {

inline bool w4_group_ok(int64_t group) { return group == 32 || group == 64 || group == 128; }

// A scale of type NPLK_DTYPE_* as it is stored, and its value: the conversion apart from the
// load, so that a load ahead of its use is not waited for (nor, in 16 bits, for its widening,
// which the compiler puts behind the load; here the load itself widens). `at` has to lie in the
// array whatever the result is used for, and the statements are volatile: the compiler may run
// an asm statement without side effects, which the headers' __ldg of 16-bit floats are, ahead
// of the condition it stands under (a scale array at the end of its memory segment faulted so).
__device__ __forceinline__ uint32_t load_scale_bits(const void *scales, int dtype, int64_t at) {
  uint32_t bits;
  if (dtype == NPLK_DTYPE_FP32) {
    asm volatile("ld.global.nc.u32 %0, [%1];"
                 : "=r"(bits)
                 : "l"(static_cast<const uint32_t *>(scales) + at));
  } else {
    asm volatile("ld.global.nc.u16 %0, [%1];"
                 : "=r"(bits)
                 : "l"(static_cast<const uint16_t *>(scales) + at));
  }
  return bits;
}
// A zero's byte, of which the low half counts: taken apart where it is used, for the same reason.
__device__ __forceinline__ uint32_t load_zero_bits(const uint8_t *zeros, int64_t at) {
  uint32_t bits;
  asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(bits) : "l"(zeros + at));
  return bits;
}
__device__ __forceinline__ float scale_value(uint32_t bits, int dtype) {
  if (dtype == NPLK_DTYPE_FP32) return __uint_as_float(bits);
  if (dtype == NPLK_DTYPE_BF16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ float load_scale(const void *scales, int dtype, int64_t at) {
  return scale_value(load_scale_bits(scales, dtype, at), dtype);
}

}  // namespace nplk
