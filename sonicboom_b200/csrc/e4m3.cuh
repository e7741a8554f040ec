// Numbers held in 8 bits (e4m3: a sign, four bits of exponent, three of mantissa; largest 448, no infinities) with a
// power-of-two scale for every block of them.
//
// A block here is one page of one head, keys and values apart.  Its scale is 2^e with the smallest e that leaves nothing
// above 448, -126 <= e <= 120.  With a power of two the division by the scale and the product with it round nothing, e4m3's
// own exponent takes the place of the bits that a finer scale would win, and going over to a larger scale later (a page
// fills up token by token) only changes exponents: numbers lose bits there only where they fall below e4m3's normal range,
// 2^-15 of the block's largest.
#pragma once

#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

constexpr int E4M3_LOWEST = -126;

// The smallest e with largest <= 448 * 2^e = 1.75 * 2^(e + 8); the argument is finite and not negative.
__device__ __forceinline__ int e4m3_exponent(float largest) {
  const uint32_t b = __float_as_uint(largest);
  return max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), E4M3_LOWEST);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }    // -126 <= e <= 127
// The exponent of a scale as it is kept (a power of two as float32).
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23 & 255) - 127; }

// The size of a value as it counts for a block's scale: infinities and NaN do not, they are stored as NaN whatever it is.
__device__ __forceinline__ float e4m3_size(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;
}
// Two values over their block's scale (given as `inverse`) to e4m3, to the nearest, ties to even; `a` in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b, float inverse) {
  a = fabsf(a) <= 3.402823466e38f ? a * inverse : NAN;
  b = fabsf(b) <= 3.402823466e38f ? b * inverse : NAN;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Two e4m3 numbers (the low 16 bits) as halves, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)v));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t v) {
  const uint32_t h = e4m3x2_to_half2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
