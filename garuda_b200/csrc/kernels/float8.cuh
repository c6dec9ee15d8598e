// Numbers in 8 bits (E4M3: four bits of exponent, three of mantissa, largest 448) with a scale per block.
//
// A block's scale is a power of two, 2^e with the smallest e >= -100 for which 448 * 2^e is at least the block's largest
// magnitude. A power of two costs E4M3 nothing (its steps are relative but for the subnormals, 2^-15 below the largest) and
// makes every change of scale exact: x / s is x with another exponent, so a value is rounded once, when it becomes a code,
// and a page whose scale grows keeps its codes but for an exponent (the subnormals are rounded again).
#pragma once

#include "common.cuh"

namespace f8 {

constexpr int BLOCK = 128;              // channels of a token, and rows by channels of a weight, that share a scale
constexpr int MIN_EXPONENT = -100, MAX_EXPONENT = 120;

// e of the block's scale 2^e. `largest` >= 0; infinity (and what overflows 448 * 2^120) takes the largest scale.
__device__ __forceinline__ int scale_exponent(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  // largest = 1.m * 2^(b - 127), 448 = 1.75 * 2^8
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, MIN_EXPONENT), MAX_EXPONENT);
}
// 2^e for e from -126 to 127
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two values as codes, the first in the lower byte; beyond 448 (infinity too) 448, NaN stays NaN.
__device__ __forceinline__ uint16_t encode2(float first, float second) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(second), "f"(first));
  return r;
}
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  return (uint32_t)encode2(a, b) | ((uint32_t)encode2(c, d) << 16);
}
// Two codes as halves (exact: every E4M3 number is one), the lower byte in the lower half.
__device__ __forceinline__ uint32_t decode2_f16(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ float2 decode2(uint32_t two) {
  const uint32_t h = decode2_f16(two);
  float2 v;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(v.x), "=f"(v.y) : "r"(h));
  return v;
}
__device__ __forceinline__ float4 decode4(uint32_t four) {
  const float2 a = decode2(four & 0xFFFFu), b = decode2(four >> 16);
  return make_float4(a.x, a.y, b.x, b.y);
}

}  // namespace f8
