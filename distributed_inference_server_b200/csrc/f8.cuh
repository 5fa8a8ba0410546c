// f8.cuh -- 8-bit floating point rows (e4m3) with a power-of-two scale for each 128 entries: what their writers and readers share.
#pragma once
#include "ptx.cuh"

namespace dis {

constexpr int kF8Block = 128;  // entries of a row, and rows of a weight, under one scale

// The scale of a block whose largest magnitude has the bits `top` (the bits of non-negative floats order as the floats do, infinities and
// NaN above): s = 2^ceil(log2(top / 448)), 448 = 1.75 * 2^8 being e4m3's largest value, so the exponent is top's less 8 and one more where its
// mantissa passes 1.75.  Not below 2^-126: 1 / s is a float.  A block that holds an infinity or a NaN has none: its scale is NaN, and so is
// every sum that takes it.  A power of two makes x / s exact: the same values whoever divides, however.
__device__ __forceinline__ float f8_scale(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}
// 1 / s of a scale that is one (2^-126 to 2^120); NaN of NaN
__device__ __forceinline__ float f8_inverse(float s) { return s == s ? __uint_as_float((254u << 23) - __float_as_uint(s)) : s; }

// Four values to e4m3, nearest with ties to even, lowest byte first
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ uint32_t f8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t f8_top4(float a, float b, float c, float d) { return max(max(f8_bits(a), f8_bits(b)), max(f8_bits(c), f8_bits(d))); }

}  // namespace dis
