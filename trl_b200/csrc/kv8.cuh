// Values of the 8-bit paged key-value cache: e4m3 codes times one power of two per (page, key head).
//
// A power of two as scale changes no code's fraction: dividing by it is exact in fp32, so a value is rounded once, to four
// significant bits, and bringing earlier rows of a page to a larger scale only rounds those that fall below e4m3's smallest
// normal number.  scale = 2^e with the smallest e that brings the largest finite magnitude within 448, held in [-100, 120]:
// 448 * 2^120 is above every finite bf16 and fp32 value, and 2^-100 keeps 1 / scale finite.
#pragma once
#include "common.cuh"

namespace trlb {

constexpr int KV8_MIN_EXP = -100, KV8_MAX_EXP = 120;

// Smallest e with amax <= 448 * 2^e.  448 = 1.75 * 2^8, so the fraction of amax decides between two exponents.
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(KV8_MAX_EXP, max(KV8_MIN_EXP, e));
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// |x| of a finite value, 0 of an infinity or NaN: those do not set a page's scale
__device__ __forceinline__ float kv8_magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.4028234663852886e38f ? a : 0.f;
}

// Two values over the scale as codes (a in the low byte).  x - x is 0 for a finite value and NaN otherwise, so infinities
// (which the conversion would saturate) and NaN are both held as NaN.
__device__ __forceinline__ uint32_t kv8_encode2(float a, float b, float inv_scale) {
  const float ya = fmaf(a, inv_scale, a - a), yb = fmaf(b, inv_scale, b - b);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(yb), "f"(ya));
  return r;
}
// The same of finite values.
__device__ __forceinline__ uint32_t kv8_encode2_finite(float a, float b, float inv_scale) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b * inv_scale), "f"(a * inv_scale));
  return r;
}
// Two codes (low byte first) as a pair of fp16, exact: fp16 has every e4m3 value.
__device__ __forceinline__ uint32_t kv8_decode2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t kv8_decode2_hi(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

}  // namespace trlb
