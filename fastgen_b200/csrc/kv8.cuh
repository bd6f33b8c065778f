// The paged cache in 8 bits: what the kernels that write it and those that read it share.
//
// A (page, key/value head) pair is a block of page * HD codes (e4m3: a sign, four bits of exponent, three of
// mantissa) with one scale 2^e, float32 [n_pages, n_kv_heads]; an entry stands for code * 2^e.
//   keys    [page, head, slot, HD]           a token's codes in a row
//   values  [page, head, slot / 4, HD, 4]    the codes of four tokens side by side
// Both operands of the second product of attention are wanted with neighbouring keys next to each other (the
// tensor core packs pairs along the dimension it sums over): four tokens' codes of one dimension are a 32-bit
// word, so a fragment is a load and two conversions, with no transposition on the way.
//
// A power of two for a scale: code * 2^e is exact in bfloat16 and float32, so what the cache stands for does not
// depend on which kernel reads it, and rounding codes again at a larger scale moves only those that leave e4m3's
// normal range (e4m3's own exponent does what the mantissa of a general scale would: its steps are relative).
// e is the smallest whole number from KV8_LOWEST on at which the block's largest magnitude is at most 448 * 2^e.
// Entries that are not finite are stored as NaN and take no part in the scale; magnitudes above 448 * 2^100
// are stored as that.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace fg_kv8 {

constexpr int KV8_LOWEST = -100, KV8_HIGHEST = 100;

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]
__device__ __forceinline__ int exponent_of_scale(float s) { return (__float_as_int(s) >> 23) - 127; }

// the smallest e with amax <= 448 * 2^e = 1.75 * 2^(8 + e), for a finite amax >= 0
__device__ __forceinline__ int scale_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
  return min(max(e, KV8_LOWEST), KV8_HIGHEST);
}

// two numbers, already over their scale, as codes: lo in bits 0-7, hi in bits 8-15
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
  uint16_t v;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(v) : "f"(hi), "f"(lo));
  return v;
}
// the two codes of the low (or high) half of a word, as half precision: exact
__device__ __forceinline__ uint32_t halves_of_low(uint32_t w) {
  uint32_t d;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t halves_of_high(uint32_t w) {
  uint32_t d;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ float2 floats_of(uint32_t halves) {
  return __half22float2(*reinterpret_cast<const __half2*>(&halves));
}

// four codes of a word rounded again after a multiplication by f (a power of two)
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float f) {
  const float2 a = floats_of(halves_of_low(w)), b = floats_of(halves_of_high(w));
  return codes_of(a.x * f, a.y * f) | (codes_of(b.x * f, b.y * f) << 16);
}

}  // namespace fg_kv8
