// Rounded quotients by a scale, for the quantisers: rint of the correctly rounded fp32
// quotient, several values at a time.
#pragma once

#include <math_constants.h>

#include "typed_io.cuh"

namespace nplk {

struct Scale {
  float value;             // as stored
  float divisor, inverse;  // value, or value * 2^64 where `lifted`, and 1 / divisor
  bool finite, lifted;
};

constexpr float kLift = 18446744073709551616.0f;  // 2^64

__device__ __forceinline__ Scale split_scale(float value) {
  Scale s;
  s.value = value;
  s.finite = s.value < CUDART_INF_F;
  s.lifted = s.value < 7.8886091e-31f;  // 2^-100
  s.divisor = s.lifted ? s.value * kLift : s.value;
  s.inverse = 1.0f / s.divisor;
  return s;
}
constexpr float kToInt = 12582912.0f;  // 1.5 * 2^23: a sum's low bits are the rounded integer

// q of a pack, in the low byte of each word: the fp32 quotient x / scale, then
// its rounding to the nearest integer.
//
// The quotient by P. Markstein's method ("Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990): with y the correctly rounded
// 1 / scale and q within one step of x / scale, q + y (x - q scale), the
// remainder exact in one fused step, is x / scale correctly rounded. x * y may be
// 1.5 steps off; one such correction brings it within one, the second is the
// theorem's. The remainder's last bit is at least 2^-48 of the scale where the
// quotient is above 1/4 (below, it rounds to 0 whatever its error): exact for
// scales from 2^-100 on; under that, x and the scale are both lifted by 2^64.
// Correcting only the products near a half instead is no faster: the coarse
// grids of 16-bit types make exact halves common, nearly every warp has one, and
// 8192 x 4096 bf16 took 23 us that way against 21.
// finite_quotients: where the scale is finite and not lifted (anything, if it is not finite).
template <typename T, int V>
__device__ __forceinline__ void finite_quotients(const float (&x)[V], const Scale &s,
                                                 uint32_t (&b)[V]) {
  if constexpr (V % 2 == 0) {
    const float2 y = make_float2(s.inverse, s.inverse), d = make_float2(-s.divisor, -s.divisor);
    const float2 one = make_float2(1.0f, 1.0f), to_int = make_float2(kToInt, kToInt);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 v = make_float2(x[j], x[j + 1]);
      float2 q = mul2(v, y);
      q = fma2(fma2(q, d, v), y, q);
      q = fma2(fma2(q, d, v), y, q);
      q = fma2(q, one, to_int);
      b[j] = __float_as_uint(q.x);
      b[j + 1] = __float_as_uint(q.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float q = x[j] * s.inverse;
      q = fmaf(fmaf(q, -s.divisor, x[j]), s.inverse, q);
      q = fmaf(fmaf(q, -s.divisor, x[j]), s.inverse, q);
      b[j] = __float_as_uint(q + kToInt);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void finite_quotients(const Pack<T, V> &p, const Scale &s,
                                                 uint32_t (&b)[V]) {
  float x[V];
  unpack(p, x);
  finite_quotients<T>(x, s, b);
}
template <typename T, int V>
__device__ __forceinline__ void quotients(const Pack<T, V> &p, const Scale &s, uint32_t (&b)[V]) {
  if (!s.finite) {
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = 0u;
    return;
  }
  float x[V];
  unpack(p, x);
  if (s.lifted) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] *= kLift;
  }
  finite_quotients<T>(x, s, b);
}

// Four low bytes as one word.
__device__ __forceinline__ uint32_t low_bytes(const uint32_t *b) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

}  // namespace nplk
