// layer_factor.cuh -- the 16 bits that bf16 tensors' factors of a backward pass are kept in.
//
// A gradient's operand is rounded to the tensors' type once it is formed; the
// factor that forms it should add little to that, and moving more than 16 bits
// of it costs where memory bounds the layer (24 bits as two planes: the gate
// of 32768 rows, 256 -> 1024, took 89 us against a floor of 41).  bf16 rounds to
// 2^-8, so f16's 2^-11 adds 1 % to a rounding's root mean square, and a power of
// two per block of 16 columns of a row brings the largest to [2^14, 2^15):
// nothing overflows, and what is 2^-28 of the largest still has its 11 bits.
//
// f16 tensors' factors are kept in f32: 16 bits have either room for more
// precision than f16's own or for its range beside a large neighbour.
#pragma once

#include "af2_device.cuh"

namespace af2 {

// A block's values v as codes; returns `e`, the biased f32 exponent of the largest.
__device__ __forceinline__ uint32_t factor_block(const float2 (&v)[8], uint32_t (&w)[8]) {
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
__device__ __forceinline__ float factor_scale(uint32_t e) { return __uint_as_float((e - 14u) << 23); }
__device__ __forceinline__ float2 factor_values(uint32_t w, float scale) { return f2mul(unpack2<__half>(w), f2(scale)); }

// Slopes: at most 1.13 in size (or NaN), so one power of two does.
__device__ __forceinline__ uint32_t slope_codes(float2 v) {
  v = f2mul(v, f2(16384.f));
  return pack_half2(v.x, v.y);
}
__device__ __forceinline__ float2 slope_values(uint32_t w) { return f2mul(unpack2<__half>(w), f2(1.f / 16384.f)); }

}  // namespace af2
