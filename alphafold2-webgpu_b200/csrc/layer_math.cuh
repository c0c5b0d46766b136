// layer_math.cuh -- the activations of the layers with learned weights and
// their slopes, in f32.
#pragma once

#include <math.h>

#include "../../include/af2cuda.h"
#include "af2_device.cuh"

namespace af2 {

// Value of the activation at z.  sigmoidf is within a few ulp (af2_device.cuh), erff CUDA's own.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == AF2_ACTIVATION_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (ACT == AF2_ACTIVATION_SIGMOID) return sigmoidf(z);
  if constexpr (ACT == AF2_ACTIVATION_SILU) return z * sigmoidf(z);
  if constexpr (ACT == AF2_ACTIVATION_GELU) return z * fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f);
  return z;
}

// Value and slope together.
//   relu:    max(z, 0);  1 where z > 0
//   sigmoid: s;          s (1 - s)
//   silu:    z s;        s (1 + z (1 - s))
//   gelu:    z Phi(z);   Phi(z) + z phi(z)
template <int ACT>
__device__ __forceinline__ void activate_slope(float z, float &value, float &slope) {
  if constexpr (ACT == AF2_ACTIVATION_NONE) {
    value = z;
    slope = 1.f;
  } else if constexpr (ACT == AF2_ACTIVATION_RELU) {
    value = z > 0.f ? z : (z != z ? z : 0.f);
    slope = z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == AF2_ACTIVATION_GELU) {
    const float cdf = fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f);
    value = z * cdf;
    slope = fmaf(z * 0.39894228040143268f, exp2f(z * z * -0.72134752044448170f), cdf);
  } else {
    const float s = sigmoidf(z);
    if constexpr (ACT == AF2_ACTIVATION_SIGMOID) {
      value = s;
      slope = s * (1.f - s);
    } else {
      value = z * s;
      slope = s * fmaf(z, 1.f - s, 1.f);
    }
  }
}

// Calls f with the activation as a compile-time constant.
template <typename F>
inline void with_activation(int activation, F &&f) {
  switch (activation) {
    case AF2_ACTIVATION_RELU: f(std::integral_constant<int, AF2_ACTIVATION_RELU>()); break;
    case AF2_ACTIVATION_SIGMOID: f(std::integral_constant<int, AF2_ACTIVATION_SIGMOID>()); break;
    case AF2_ACTIVATION_SILU: f(std::integral_constant<int, AF2_ACTIVATION_SILU>()); break;
    case AF2_ACTIVATION_GELU: f(std::integral_constant<int, AF2_ACTIVATION_GELU>()); break;
    default: f(std::integral_constant<int, AF2_ACTIVATION_NONE>()); break;
  }
}

// Calls f with a null pointer of the element type.
template <typename F>
inline void with_element(int dtype, F &&f) {
  if (dtype == AF2_F16)
    f(static_cast<__half *>(nullptr));
  else if (dtype == AF2_BF16)
    f(static_cast<__nv_bfloat16 *>(nullptr));
  else
    f(static_cast<float *>(nullptr));
}

}  // namespace af2
