// Activations over small register arrays, for epilogues whose result type is
// known: the code is chosen once per array instead of once per value.
#pragma once

#include <type_traits>

#include "activation_grad.cuh"
#include "nplk_device.cuh"

namespace nplk {

// The activations that no array form below inlines: one call per value keeps
// the epilogues small.
static __device__ __noinline__ float act_call(float x, int act, float alpha) {
  return apply_act(x, act, alpha);
}

// v[j] = act(v[j]), results to be stored as T. fp32 results take the formulas
// of apply_act as they are. 16-bit results take the fast exponential and
// quotient for swish and GELU (0.5 x (1 + tanh u) = x / (1 + exp(-2u))): their
// relative error, at most a few 2^-22 for |x| <= 16 (__expf: 2 + 1.2 |x| steps
// of 2^-23; below x = -16 the value itself is under 2e-6), is below a hundredth
// of the half step of 2^-11 (fp16) or 2^-8 (bf16) that the store rounds by.
template <typename T, int V>
__device__ __forceinline__ void act_array(float (&v)[V], int act, float alpha) {
  constexpr bool kFast = !std::is_same<T, float>::value;
  switch (act) {
    case 0:
      return;
    case 1:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
      return;
    case 5:
      if (kFast) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = v[j];
          const float u2 = x * fmaf(-2.0f * 0.7978845608f * 0.044715f, x * x, -2.0f * 0.7978845608f);
          v[j] = __fdividef(x, 1.0f + __expf(u2));
        }
        return;
      }
      break;
    case 6:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = v[j];
        v[j] = kFast ? __fdividef(x, 1.0f + __expf(-x)) : apply_act(x, 6, alpha);
      }
      return;
    default:
      break;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = act_call(v[j], act, alpha);
}

static __device__ __noinline__ float act_slope_call(float x, int act, float alpha) {
  return act_slope(x, act, alpha);
}

// v[j] = act'(v[j]), for gradients stored as T; 16-bit results as above.
template <typename T, int V>
__device__ __forceinline__ void act_slope_array(float (&v)[V], int act, float alpha) {
  constexpr bool kFast = !std::is_same<T, float>::value;
  switch (act) {
    case 0:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 1.0f;
      return;
    case 1:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] > 0.0f ? 1.0f : 0.0f;
      return;
    case 5:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = v[j], x2 = x * x;
        const float c = 2.0f * 0.7978845608f, k = c * 0.044715f;
        if (kFast) {
          const float s = __fdividef(1.0f, 1.0f + __expf(-x * fmaf(k, x2, c)));
          v[j] = s + x * s * (1.0f - s) * fmaf(3.0f * k, x2, c);
        } else {
          v[j] = act_slope(x, 5, alpha);
        }
      }
      return;
    case 6:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = v[j];
        const float s = kFast ? __fdividef(1.0f, 1.0f + __expf(-x)) : 1.0f / (1.0f + expf(-x));
        v[j] = s * fmaf(x, 1.0f - s, 1.0f);
      }
      return;
    default:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_slope_call(v[j], act, alpha);
      return;
  }
}

}  // namespace nplk
