// Derivatives of the activations in nplk_device.cuh, at their input.
#pragma once

#include "nplk_device.cuh"

namespace nplk {

// act'(x) for codes 0..10 (npl_activation_t). ReLU, LeakyReLU, ELU and SELU
// take the left-hand value at 0, ReLU6 is 0 at both bends.
__device__ __forceinline__ float act_slope(float x, int act, float alpha) {
  switch (act) {
    case 1:
      return x > 0.0f ? 1.0f : 0.0f;
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
    case 5: {  // y = x * s with s = sigmoid(2u) = (1 + tanh(u)) / 2, u = c (x + a x^3)
      const float x2 = x * x;
      const float s = 1.0f / (1.0f + expf(-2.0f * 0.7978845608f * x * (1.0f + 0.044715f * x2)));
      return s + 2.0f * x * s * (1.0f - s) * 0.7978845608f * (1.0f + 3.0f * 0.044715f * x2);
    }
    case 6: {
      const float s = 1.0f / (1.0f + expf(-x));
      return s * (1.0f + x * (1.0f - s));
    }
    case 7:
      return x > 0.0f ? 1.0f : alpha;
    case 8:
      return x > 0.0f ? 1.0f : expf(x);
    case 9:
      return 1.05070098f * (x > 0.0f ? 1.0f : 1.67326324f * expf(x));
    case 10:
      return 1.0f / (1.0f + expf(-x));
    default:
      return 1.0f;
  }
}

}  // namespace nplk
