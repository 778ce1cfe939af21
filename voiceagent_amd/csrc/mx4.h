// MXFP4 KV pools: OCP MX e2m1 codes, two to a byte (the even element in the
// low half), with one e8m0 scale byte for each 32 elements of a row.
//
// A code c with scale byte s stands for grid(c) 2^(s - 127), grid = 0, 1/2, 1,
// 3/2, 2, 3, 4, 6 and their negatives.  Quantising a group takes the smallest
// exponent e with max |x| < 7 2^e, so the largest element is off by at most
// 2^e (7 2^e rounds down to 6 2^e, and 6 to 8 2^e in the next binade's
// grid), half the grid's widest step; with the usual floor(log2 max) - 2 an
// element just below 8 2^e would be off by two.  e is kept where 6 2^e and
// 2^e / 2 are representable in the rows' type (bf16: -125 .. 125, f16:
// -23 .. 13), so every value converts back to that type exactly; infinities
// saturate.  A group that holds a NaN gets scale 255 and reads as NaN.
// Codes are rounded to nearest, ties to even, by gfx950's conversion, which
// divides by the scale without rounding first and saturates at 6.
#pragma once

#include "common.h"

namespace va {

constexpr int kMx4Group = 32;  // elements per scale

// Scale bytes a store may write, by row type (see above).
template <typename ET>
struct Mx4Range;
template <>
struct Mx4Range<BF16> {
  static constexpr int lo = 2, hi = 252;
};
template <>
struct Mx4Range<F16> {
  static constexpr int lo = 104, hi = 140;
};

// Largest |element| bits of 8 16-bit elements.  The bits of a magnitude order
// as the magnitudes do, infinity above the finite values and NaN above it.
__device__ inline uint32_t mx4_absmax8(uint4 u) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  auto mag = [](uint32_t x) { return __builtin_bit_cast(u16x2, x & 0x7fff7fffu); };
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(u.x), mag(u.y)),
                                            __builtin_elementwise_max(mag(u.z), mag(u.w)));
  return m.x > m.y ? m.x : m.y;
}

// Largest of the values of four neighbouring lanes.
__device__ inline uint32_t quad_max(uint32_t x) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppQuadXor1, 0xF, 0xF, false);
  x = x > a ? x : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppQuadXor2, 0xF, 0xF, false);
  return x > b ? x : b;
}

// Scale byte of a group whose largest magnitude has these bits.
template <typename ET>
__device__ inline uint32_t mx4_scale(uint32_t mag) {
  const uint32_t bits = ET::kIsBF16
                            ? mag << 16
                            : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)mag));
  // Adding a quarter to the mantissa carries at 1.75 2^E, that is at 7 2^e.
  int e = (int)((bits + 0x200000u) >> 23) - 2;
  e = e < Mx4Range<ET>::lo ? Mx4Range<ET>::lo : (e > Mx4Range<ET>::hi ? Mx4Range<ET>::hi : e);
  return bits > 0x7f800000u ? 255u : (uint32_t)e;
}

// 8 elements (element i at half i of u) as 8 codes, element i in nibble i; a
// NaN group's codes are 0.
template <typename ET>
__device__ inline uint32_t mx4_codes8(uint4 u, uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  float f[8];
  ET::unpack(u, f);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], s, 3);
  return scale == 255u ? 0u : w;
}

// Codes 2 B and 2 B + 1 of a word as two elements of ET, the first in the low
// half; scale is a power of two (or NaN), as a float.
template <typename ET, int B>
__device__ inline uint32_t mx4_pair(uint32_t codes, float scale) {
  if constexpr (ET::kIsBF16)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B));
}

// 8 codes as 8 elements of ET.
template <typename ET>
__device__ inline uint4 mx4_values8(uint32_t codes, uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  return make_uint4(mx4_pair<ET, 0>(codes, s), mx4_pair<ET, 1>(codes, s),
                    mx4_pair<ET, 2>(codes, s), mx4_pair<ET, 3>(codes, s));
}

// Host checks of a pool's scale arrays that every entry point makes, for rows
// of head_dim elements: rows of scales are read as single words.
int check_mx4(const char* fn, const va_kv_pool& pool, const va_mx4_scales* sc, int head_dim);

}  // namespace va
