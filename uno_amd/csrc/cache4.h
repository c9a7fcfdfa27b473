// Cache rows in 4 bits: E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) with one E8M0 scale, 2^(byte - 127), to GROUP4
// consecutive elements. A row of D elements is D / 2 bytes of codes (the even element in the low half) and D / GROUP4 scale bytes;
// codes and scales lie in tensors of their own, [batch, nk, max_len, ..], contiguous.
//
// The scale is the least power of two of which a group's largest magnitude is less than seven: that magnitude then rounds to six at
// most, and a scale twice as large would give the largest magnitudes the same numbers and the others coarser ones. Scaling is exact
// and the rounding is to the nearest number, ties to the even code, so that a row's codes are a function of its elements, whatever
// their type. Every number is exact in bf16 (the least scale is 2^-125, half of which is no subnormal; the largest 2^125, six of which
// are finite). A group that holds an infinity or NaN has scale byte 255, which makes its elements NaN.
//
// The conversions (v_cvt_scalef32_pk_*) read the scale's exponent alone, and make NaN of byte 255.
#pragma once
#include "common.h"

constexpr int GROUP4 = 32, SCALE4_MIN = 2, SCALE4_MAX = 252, SCALE4_NAN = 255;

struct Row4 { const uint8_t *codes, *scales; };

__device__ __forceinline__ float scale4(uint32_t byte) { return __uint_as_float(byte << 23); }

// Elements 2 BYTE and 2 BYTE + 1 of eight codes as bf16.
template <int BYTE> __device__ __forceinline__ uint32_t pair4(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
}

__device__ __forceinline__ float value4(Row4 r, int d) {
  const uint32_t u = pair4<0>(r.codes[d / 2], scale4(r.scales[d / GROUP4]));
  return __uint_as_float(d % 2 ? u & 0xffff0000u : u << 16);
}

// The scale byte of a group whose largest magnitude is `top` (NaN or infinite: a number that is no number).
__device__ __forceinline__ uint32_t scale4_of(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u >= 0x7f800000u) return SCALE4_NAN;
  // top < 7 * 2^(e - 127): with top = m 2^x, m in [1, 2), x - 2 for m < 1.75, else x - 1
  const int e = (int)(u >> 23) - ((u & 0x7fffffu) < 0x600000u ? 2 : 1);
  return (uint32_t)min(max(e, SCALE4_MIN), SCALE4_MAX);
}

// Two elements appended as codes to byte BYTE of `codes`; magnitudes above six scales become six.
template <int BYTE> __device__ __forceinline__ uint32_t codes4(uint32_t codes, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, scale, BYTE);
}
