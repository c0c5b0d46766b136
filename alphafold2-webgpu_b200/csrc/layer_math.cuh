// layer_math.cuh -- the activations of the layers with learned weights and
// their slopes, in f32.
//
//   relu:    max(z, 0);  1 where z > 0
//   sigmoid: s;          s (1 - s)            s = 1 / (1 + e^-z), 1 - s = e^-z s
//   silu:    z s;        s (1 + z (1 - s))
//   gelu:    z Phi(z);   Phi(z) + z phi(z)    Phi, phi of the standard normal
//
// Two elements at a time, because the epilogues that call it are bound by the
// multi-function unit and by issue slots.  Two forms: FAST = false, for f32
// tensors, within some ten units of f32's last place, on the negative side too;
// FAST = true, for 16-bit ones, relative error below 2^-16 where the value
// matters to them.
//   - f32: an exponential's argument is a rounded product, whose error grows with it
//     (|z| 2^-24 of e^-z, z^2 2^-24 of e^(-z^2 / 2)): fma gives the product's
//     rest, and the exponential is multiplied by 1 + ln 2 of that.
//   - FAST: two sigmoids share one reciprocal: with d = 1 + e^-z, 1 / d0 =
//     d1 / (d0 d1).  The exponential is held below 2^63 so that the product cannot
//     overflow, and 2^-62 is taken off the sigmoid, with 0 as the least: far out it
//     is 0, not the bound, which a z of the type's lowest value would make large of.
//     What that takes off a sigmoid is 2^-16 of it at z = -32.
//   - Phi(-u) = e^(-u^2 / 2) t Q(t), t = 1 / (1 + c u), u >= 0: the form of
//     Hastings' approximations, Q fitted to Phi(-u) e^(u^2 / 2) / t on u in [0, 14]
//     for the least largest relative error (degree 5, c = 0.31: 4.7e-6; degree 8,
//     c = 0.265: 1.2e-8).  No cancellation for z < 0, and the exponential serves
//     the slope too.
#pragma once

#include "../../include/af2cuda.h"
#include "af2_device.cuh"

namespace af2 {

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The sigmoids with the denominators d.
__device__ __forceinline__ float2 shared_reciprocal(float2 d) {
  const float r = rcp_approx(d.x * d.y);
  return make_float2(__saturatef(fmaf(r, d.y, -0x1p-62f)), __saturatef(fmaf(r, d.x, -0x1p-62f)));
}
// The sigmoids of two values; a NaN gives 0 (its product with z is NaN again).
__device__ __forceinline__ float2 sigmoid2_fast(float2 z) {
  const float2 x = f2mul(z, f2(-1.4426950408889634f));
  return shared_reciprocal(f2add(make_float2(ex2_approx(fminf(x.x, 63.f)), ex2_approx(fminf(x.y, 63.f))), f2(1.f)));
}

// 2^(x - over), `over` within x's rounding (none where x is out of f32's range of powers).
__device__ __forceinline__ float ex2_less(float x, float over) {
  return ex2_approx(x) * fmaf(fabsf(x) < 160.f ? over : 0.f, -0.69314718f, 1.f);
}
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.9259630e-8f;  // and what its rounding left

// e^-z of two values.
template <bool FAST>
__device__ __forceinline__ float2 exp_of_minus(float2 z) {
  const float2 x = f2mul(z, f2(-kLog2e));
  if constexpr (FAST) return make_float2(ex2_approx(x.x), ex2_approx(x.y));
  const float2 over = f2fma(z, f2(kLog2eRest), f2fma(z, f2(kLog2e), x));
  return make_float2(ex2_less(x.x, over.x), ex2_less(x.y, over.y));
}

// The sigmoids of two values to f32's accuracy.
__device__ __forceinline__ float2 sigmoid2_f32(float2 z) {
  const float2 e = exp_of_minus<false>(z);
  return make_float2(rcp_approx(1.f + e.x), rcp_approx(1.f + e.y));
}

// Phi and, for the slope, e^(-z^2 / 2).
template <bool FAST>
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2 &e) {
  const float2 square = f2mul(z, z), arg = f2mul(square, f2(-kLog2e / 2));
  if constexpr (FAST) {
    e = make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
  } else {
    float2 over = f2fma(square, f2(kLog2e / 2), arg);
    over = f2fma(square, f2(kLog2eRest / 2), over);
    over = f2fma(make_float2(fmaf(z.x, z.x, -square.x), fmaf(z.y, z.y, -square.y)), f2(kLog2e / 2), over);
    e = make_float2(ex2_less(arg.x, over.x), ex2_less(arg.y, over.y));
  }
  const float2 d = f2fma(make_float2(fabsf(z.x), fabsf(z.y)), f2(FAST ? 0.31f : 0.265f), f2(1.f));
  const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  float2 q;
  if constexpr (FAST) {
    q = f2fma(f2(-0.07392890751361847f), t, f2(0.1804496943950653f));
    q = f2fma(q, t, f2(0.015745392069220543f));
    q = f2fma(q, t, f2(0.13342945277690887f));
    q = f2fma(q, t, f2(0.12044135481119156f));
    q = f2fma(q, t, f2(0.12386069446802139f));
  } else {
    q = f2fma(f2(0.030820608139038086f), t, f2(-0.14422746002674103f));
    q = f2fma(q, t, f2(0.21781262755393982f));
    q = f2fma(q, t, f2(-0.11636003851890564f));
    q = f2fma(q, t, f2(0.13795138895511627f));
    q = f2fma(q, t, f2(0.06031380966305733f));
    q = f2fma(q, t, f2(0.10270080715417862f));
    q = f2fma(q, t, f2(0.10524668544530869f));
    q = f2fma(q, t, f2(0.10574156045913696f));
  }
  const float2 w = f2mul(f2mul(q, t), e);
  return make_float2(z.x < 0.f ? w.x : 1.f - w.x, z.y < 0.f ? w.y : 1.f - w.y);
}

__device__ __forceinline__ float relu(float z) { return z > 0.f ? z : (z != z ? z : 0.f); }

// Values at two places.
template <int ACT, bool FAST>
__device__ __forceinline__ float2 activate2(float2 z) {
  if constexpr (ACT == AF2_ACTIVATION_RELU) return make_float2(relu(z.x), relu(z.y));
  if constexpr (ACT == AF2_ACTIVATION_SIGMOID)
    return FAST ? make_float2(sigmoidf(z.x), sigmoidf(z.y)) : sigmoid2_f32(z);
  if constexpr (ACT == AF2_ACTIVATION_SILU) return f2mul(z, FAST ? sigmoid2_fast(z) : sigmoid2_f32(z));
  if constexpr (ACT == AF2_ACTIVATION_GELU) {
    float2 e;
    return f2mul(z, normal_cdf2<FAST>(z, e));
  }
  return z;
}

// Values and slopes at two places.
template <int ACT, bool FAST>
__device__ __forceinline__ void activate_slope2(float2 z, float2 &value, float2 &slope) {
  if constexpr (ACT == AF2_ACTIVATION_NONE) {
    value = z;
    slope = f2(1.f);
  } else if constexpr (ACT == AF2_ACTIVATION_RELU) {
    value = make_float2(relu(z.x), relu(z.y));
    slope = make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
  } else if constexpr (ACT == AF2_ACTIVATION_GELU) {
    float2 e;
    const float2 cdf = normal_cdf2<FAST>(z, e);
    value = f2mul(z, cdf);
    slope = f2fma(f2mul(z, f2(0.39894228040143268f)), e, cdf);
  } else {
    if constexpr (ACT == AF2_ACTIVATION_SIGMOID) {
      const float2 e = exp_of_minus<FAST>(z);
      value = make_float2(rcp_approx(1.f + e.x), rcp_approx(1.f + e.y));
      // 1 - s, which cancels where z is large, is e^-z s
      slope = f2mul(value, make_float2(z.x > 0.f ? e.x * value.x : 1.f - value.x,
                                       z.y > 0.f ? e.y * value.y : 1.f - value.y));
    } else {
      const float2 s = FAST ? sigmoid2_fast(z) : sigmoid2_f32(z);
      value = f2mul(z, s);
      slope = f2mul(s, f2fma(z, f2fma(s, f2(-1.f), f2(1.f)), f2(1.f)));
    }
  }
}

// Calls f with the activation as a compile-time constant (host and device).
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int activation, F &&f) {
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

// The three bf16 terms of eight f32, x = t0 + t1 + t2 exactly (but for what is below f32's smallest
// normal number): the upper 16 bits of x, of what that leaves, and of what is then left.  Cutting
// instead of rounding costs an and and a subtraction a term, and no finite x can overflow.
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&t)[3]) {
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      w[k][i] = __byte_perm(a, b, 0x7632);
      if (k < 2) {
        a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xffff0000u));
        b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xffff0000u));
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) t[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}

}  // namespace af2
