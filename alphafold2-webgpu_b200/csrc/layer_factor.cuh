// layer_factor.cuh -- the 16 bits that the factors of a backward pass are kept in.
//
// A gradient's operand is rounded to the tensors' type once it is formed; the
// factor that forms it should add little to that, and moving more than 16 bits
// of it costs where memory bounds the layer (24 bits as two planes: the gate
// of 32768 rows, 256 -> 1024, took 89 us against a floor of 41).  So the format
// follows the type:
//
//   bf16 (rounds to 2^-8): f16, to 2^-11, scaled by a power of two so that the
//   largest of a block is in [2^14, 2^15): nothing overflows, and what is
//   2^-28 of the largest still has its 11 bits.
//
//   f16 (rounds to 2^-11): a dense layer's slopes are kept in f32 (16 bits hold
//   either f16's precision or its range).  The gated transition's factors: sign, 3 bits of exponent, 12 of mantissa, to 2^-13,
//   scaled so that the largest has exponent 6 of 7 (rounding may carry to 7):
//   full precision for six binades, below them steps of 2^-17 of the largest's
//   binade, as f16 itself ends 2^-14 below one.  In f32 terms: the value times
//   a power of two that brings it to the bottom of f32's range, whose gradual
//   underflow does the rest, and bits 25..11 of that.
//
// A block is 16 columns of a row, `e` the biased f32 exponent of its largest.
#pragma once

#include "af2_device.cuh"

namespace af2 {

template <typename T>
struct Factor;

template <>
struct Factor<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t block(const float2 (&v)[8], uint32_t (&w)[8]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
    const uint32_t e = max(__float_as_uint(most) >> 23, 15u);  // below 2^-112 the scale stays 2^126
    const float2 scale = f2(__uint_as_float((268u - e) << 23));  // an infinity or a NaN stays one
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = f2mul(v[i], scale);
      w[i] = pack_half2(x.x, x.y);
    }
    return e;
  }
  static __device__ __forceinline__ float scale(uint32_t e) { return __uint_as_float((e - 14u) << 23); }
  static __device__ __forceinline__ float2 value(uint32_t w, float scale) {
    return f2mul(unpack2<__half>(w), f2(scale));
  }
  // A slope: at most 1.13 in size (or NaN).
  static __device__ __forceinline__ uint32_t slope(float2 v) {
    v = f2mul(v, f2(16384.f));
    return pack_half2(v.x, v.y);
  }
  static __device__ __forceinline__ float2 slope_value(uint32_t w) {
    return f2mul(unpack2<__half>(w), f2(1.f / 16384.f));
  }
};

template <>
struct Factor<__half> {
  static constexpr float kDown = 0x1p-121f, kUp = 0x1p121f;  // exponent 127 to 6 and back
  // Two values of exponent at most 6 (as f32) as two codes.
  static __device__ __forceinline__ uint32_t codes(float2 v) {
    const uint32_t a = __float_as_uint(v.x) + 0x400u, b = __float_as_uint(v.y) + 0x400u;
    return ((a >> 11) & 0x7fffu) | ((a >> 16) & 0x8000u) | ((b << 5) & 0x7fff0000u) | (b & 0x80000000u);
  }
  static __device__ __forceinline__ float2 decode(uint32_t w) {
    const float2 v = make_float2(__uint_as_float(((w << 11) & 0x03fff800u) | ((w << 16) & 0x80000000u)),
                                 __uint_as_float(((w >> 5) & 0x03fff800u) | (w & 0x80000000u)));
    return f2mul(v, f2(kUp));
  }
  static __device__ __forceinline__ uint32_t block(const float2 (&v)[8], uint32_t (&w)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      most = max(most, max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu));
    // 254 and 255 (2^127 and more, infinities, NaNs) make the block NaN: f16 tensors hold none of them
    const uint32_t e = max(most >> 23, 1u);
    const float2 scale = f2(__uint_as_float((254u - min(e, 253u)) << 23));
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = codes(f2mul(f2mul(v[i], scale), f2(kDown)));
    return e;
  }
  static __device__ __forceinline__ float scale(uint32_t e) { return __uint_as_float(e < 254u ? e << 23 : 0x7fffffffu); }
  static __device__ __forceinline__ float2 value(uint32_t w, float scale) { return f2mul(decode(w), f2(scale)); }
};

}  // namespace af2
