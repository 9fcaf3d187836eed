// Activations over small register arrays, for epilogues whose result type is
// known: the code is chosen once per array instead of once per value.
#pragma once

#include <type_traits>

#include "nplk_device.cuh"
#include "typed_io.cuh"

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

// The larger of x and `low`; a NaN stays.
__device__ __forceinline__ float at_least(float x, float low) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
  return r;
}
__device__ __forceinline__ float2 at_least(float2 x, float low) {
  return make_float2(at_least(x.x, low), at_least(x.y, low));
}

// 1 / (1 + exp(-x)) of two values that are at least -42, exp(-x) as 2^t with
// t = -x log2 e.
//
// With kShare one reciprocal serves both: 1 / a = b (1 / ab), ab below 2^122. The
// exponential and reciprocal units (16 a clock and SM) are near the bound of the
// norm: two per value are 4.6 us for 10.5 M values, whose 42 MB move in 6.4 us (4 x
// 4096 x 320 fp16: 11.9 us against 12.5; 4 x 16384 x 512 bf16: 43.6 against 44.9).
// The gradient, with more other work a value, is 3% faster with two. A NaN would
// make both results NaN then: the caller passes fmaxf(x, limit), which drops it. A
// result's last bit depends on its partner.
// kFine = false: 2^t and the reciprocal are within 2^-22 relative and t rounds by
// |t| 2^-24: below a hundredth of the half steps of fp16 (2^-11) and bf16 (2^-8).
// kFine = true, for fp32 results: one Newton step on the reciprocal; the error
// left is the exponential's, at most s (1 - s) (2^-22 + |x| 2^-24), and three
// roundings. The library's expf and division took 39 instructions a value in the
// fp32 norm, 70 us of 134 MB read and written that way against 41.
template <bool kFine, bool kShare>
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  constexpr float kLog2e = 1.44269504f;
  const float2 t = mul2(x, both(-kLog2e));
  const float2 d = add2(make_float2(exp2_approx(t.x), exp2_approx(t.y)), both(1.0f));
  if (!kShare) {
    const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    return kFine ? fma2(r, fma2(make_float2(-d.x, -d.y), r, both(1.0f)), r) : r;
  }
  const float ab = d.x * d.y;
  float r = rcp_approx(ab);
  if (kFine) r = fmaf(r, fmaf(-ab, r, 1.0f), r);
  return mul2(make_float2(d.y, d.x), both(r));
}

// The two-value steps of the array forms below: f(pair) for each pair, a lone
// value as both halves of one.
template <int V, typename F>
__device__ __forceinline__ void by_pairs(float (&v)[V], F f) {
  if constexpr (V == 1) {
    v[0] = f(make_float2(v[0], v[0])).x;
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 r = f(make_float2(v[j], v[j + 1]));
      v[j] = r.x;
      v[j + 1] = r.y;
    }
  }
}

// Below these the sigmoid of x, and of GELU's 2 u, is under 2^-58: x stops there, so
// that x * sigmoid stays under 4e-17 and nothing overflows, -infinity included.
constexpr float kSwishLow = -41.5f, kGeluLow = -7.4f;

// v[j] = act(v[j]), results to be stored as T. GELU in the form
// 0.5 x (1 + tanh u) = x * sigmoid(2 u), u = c (x + a x^3). kShare as above; without it
// v[j] depends on its own input alone.
template <typename T, bool kShare, int V>
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
      by_pairs(v, [](float2 x) {
        constexpr float c = 2.0f * 0.7978845608f;
        x = at_least(x, kGeluLow);
        const float2 w =
            kShare ? make_float2(fmaxf(x.x, kGeluLow), fmaxf(x.y, kGeluLow)) : x;
        const float2 u = mul2(w, fma2(both(c * 0.044715f), mul2(w, w), both(c)));
        return mul2(x, sigmoid2<kFine, kShare>(u));
      });
      return;
    case 6:
      by_pairs(v, [](float2 x) {
        x = at_least(x, kSwishLow);
        const float2 w =
            kShare ? make_float2(fmaxf(x.x, kSwishLow), fmaxf(x.y, kSwishLow)) : x;
        return mul2(x, sigmoid2<kFine, kShare>(w));
      });
      return;
    default:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_call(v[j], act, alpha);
      return;
  }
}

// act'(x) of the activations that act_slope_array has no form of its own for: codes 2, 3,
// 4 and 7..10. LeakyReLU, ELU and SELU take the left-hand value at 0, ReLU6 is 0 at both
// bends.
static __device__ __noinline__ float act_slope_call(float x, int act, float alpha) {
  switch (act) {
    case 2:
      return x > 0.0f && x < 6.0f ? 1.0f : 0.0f;
    case 3: {
      const float t = tanhf(x);
      return 1.0f - t * t;
    }
    case 4: {
      const float s = 1.0f / (1.0f + expf(-x));
      return s * (1.0f - s);
    }
    case 7:
      return x > 0.0f ? 1.0f : alpha;
    case 8:
      return x > 0.0f ? 1.0f : expf(x);
    case 9:
      return 1.05070098f * (x > 0.0f ? 1.0f : 1.67326324f * expf(x));
    default:  // 10
      return 1.0f / (1.0f + expf(-x));
  }
}

// v[j] = act'(v[j]), for gradients stored as T; ReLU's left-hand value at 0.
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
      by_pairs(v, [](float2 x) {
        constexpr float c = 2.0f * 0.7978845608f, k = c * 0.044715f;
        x = at_least(x, kGeluLow);
        x = make_float2(-at_least(-x.x, -30.0f), -at_least(-x.y, -30.0f));  // the slope is 1 there
        const float2 x2 = mul2(x, x);
        const float2 s = sigmoid2<kFine, false>(mul2(x, fma2(both(k), x2, both(c))));
        const float2 du = fma2(both(3.0f * k), x2, both(c));  // of u = c x + k x^3
        const float2 t = mul2(mul2(x, du), fma2(s, both(-1.0f), both(1.0f)));
        return fma2(s, t, s);  // s + x s (1 - s) u'
      });
      return;
    case 6:
      by_pairs(v, [](float2 x) {
        x = at_least(x, kSwishLow);
        const float2 s = sigmoid2<kFine, false>(x);
        return mul2(s, fma2(x, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
      });
      return;
    default:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_slope_call(v[j], act, alpha);
      return;
  }
}

}  // namespace nplk
