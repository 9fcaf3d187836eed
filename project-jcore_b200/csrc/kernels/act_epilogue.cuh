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

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / (1 + exp(-x)), exp(-x) as 2^(-x log2 e), for x multiplied on afterwards
// (x NaN then gives NaN, x = -inf NaN as the plain formula does).
// kFine = false: 2^t and the reciprocal are within 2^-22 relative and t rounds by
// |t| 2^-24: below a hundredth of the half steps of fp16 (2^-11) and bf16 (2^-8).
// kFine = true, for fp32 results: one Newton step on the reciprocal; the error
// left is the exponential's, at most s (1 - s) (2^-22 + |x| 2^-24). t stops at 126
// so that 1 + 2^t stays finite in the step.
// The library's expf and division took 39 instructions a value in the fp32
// norm, 70 us of 134 MB read and written that way.
template <bool kFine>
__device__ __forceinline__ float sigmoid(float x) {
  constexpr float kLog2e = 1.44269504f;
  if (!kFine) return rcp_approx(1.0f + exp2_approx(-kLog2e * x));
  const float d = 1.0f + exp2_approx(fminf(-kLog2e * x, 126.0f));
  const float r = rcp_approx(d);
  return fmaf(r, fmaf(-d, r, 1.0f), r);
}

// v[j] = act(v[j]), results to be stored as T. GELU in the form
// 0.5 x (1 + tanh u) = x * sigmoid(2 u), u = c (x + a x^3).
template <typename T, int V>
__device__ __forceinline__ void act_array(float (&v)[V], int act, float alpha) {
  constexpr bool kFine = std::is_same<T, float>::value;
  switch (act) {
    case 0:
      return;
    case 1:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
      return;
    case 5:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = v[j], c = 2.0f * 0.7978845608f;
        v[j] = x * sigmoid<kFine>(x * fmaf(c * 0.044715f, x * x, c));
      }
      return;
    case 6:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= sigmoid<kFine>(v[j]);
      return;
    default:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_call(v[j], act, alpha);
      return;
  }
}

static __device__ __noinline__ float act_slope_call(float x, int act, float alpha) {
  return act_slope(x, act, alpha);
}

// v[j] = act'(v[j]), for gradients stored as T; 16-bit results as above.
template <typename T, int V>
__device__ __forceinline__ void act_slope_array(float (&v)[V], int act, float alpha) {
  constexpr bool kFine = std::is_same<T, float>::value;
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
        const float x = v[j], x2 = x * x, c = 2.0f * 0.7978845608f, k = c * 0.044715f;
        const float s = sigmoid<kFine>(x * fmaf(k, x2, c));
        v[j] = s + x * s * (1.0f - s) * fmaf(3.0f * k, x2, c);
      }
      return;
    case 6:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float s = sigmoid<kFine>(v[j]);
        v[j] = s * fmaf(v[j], 1.0f - s, 1.0f);
      }
      return;
    default:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_slope_call(v[j], act, alpha);
      return;
  }
}

}  // namespace nplk
