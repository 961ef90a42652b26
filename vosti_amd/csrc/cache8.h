// Keys and values in 8 bits: what the kernels that write and read such a cache share.
//
//   keys    [pages, nkv, P, d]   and   values [pages, nkv, d, P]   e4m3 (four binary digits, largest 448, no infinity)
//   scales  [pages, nkv, 2]      32-bit: what a page's entries of a head stand in, keys' and values'.  Powers of two, 2^CACHE8_LOWEST at least.
//
// An entry stands for its value times its page's and head's scale.  The scale is the least power of two with which every entry that the
// page has been given so far is at most 448.  A power of two, and not the quotient that would use the range to its end, because an entry's four digits
// then do not depend on its neighbours: a page whose scale grows as tokens arrive holds what it would hold had it known them all, but for entries
// below 2^-14 of its largest, and the scale goes into the exponent of the number that a product takes, with no rounding.
#pragma once
#include "common.h"

#define CACHE8_LOWEST (-64)
#define CACHE8_MIN_PAGE 16       // keys: what a lane reads of a value row at once
#define CACHE8_MAX_PAGE 256

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }            // -126 .. 127
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__builtin_bit_cast(uint32_t, scale) >> 23 & 255) - 127; }

// The least e with |x| <= 448 * 2^e = 1.75 * 2^(e + 8); CACHE8_LOWEST at least, and for what is not finite.
__device__ __forceinline__ int least_exponent(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  const int e = (int)(u >> 23) - 127;
  return e > 127 ? CACHE8_LOWEST : max(CACHE8_LOWEST, e - 8 + ((u & 0x7fffffu) > 0x600000u));
}
// A 64-bit number in 32 bits, the last of them set where bits were lost: whatever is rounded to fewer digits from there (four) is rounded as from all 53, for a number that is no tie, or
// that is above a limit of few digits, remains so.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = (float)x;
  const double back = (double)f;
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  if (back != x && (u >> 23 & 255) != 255) u = (u - (fabs(back) > fabs(x) ? 1u : 0u)) | 1u;
  return __builtin_bit_cast(float, u);
}
// What a conversion to e4m3 is given for the entry x of a page with the scale 2^e: x / 2^e, and NaN for what is not finite (e4m3 has no infinity, and a
// clipped one would go unnoticed).
__device__ __forceinline__ float entry_of(float x, int e) {
  return (__builtin_bit_cast(uint32_t, x) >> 23 & 255) == 255 ? NAN : x * pow2f(-e);
}

// Four e4m3 values of four numbers, the first in the lowest byte.
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// Bytes 0 and 1 (2 and 3) of x as numbers times 2^(scale's exponent).
template <bool HI>
__device__ __forceinline__ f32x2 from_fp8x2(uint32_t x, float scale) {
  const auto r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, HI);
  return f32x2{r[0], r[1]};
}
