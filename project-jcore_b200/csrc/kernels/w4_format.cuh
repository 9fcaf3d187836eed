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
// load, so that a load ahead of its use is not waited for. `at` has to lie in the array
// whatever the result is used for: the headers' __ldg of __half and __nv_bfloat16 are asm
// statements without side effects, which the compiler may run ahead of the condition they
// stand under (a scale array at the end of its memory segment faulted so). The integer
// __ldg is no such asm.
__device__ __forceinline__ uint32_t load_scale_bits(const void *scales, int dtype, int64_t at) {
  return dtype == NPLK_DTYPE_FP32 ? __ldg(static_cast<const unsigned int *>(scales) + at)
                                  : __ldg(static_cast<const unsigned short *>(scales) + at);
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
