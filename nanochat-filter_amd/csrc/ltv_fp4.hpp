// Values in 4 bits: codes of one sign, two exponent and one mantissa bit (0, 0.5, 1,
// 1.5, 2, 3, 4, 6), and for 32 of them one byte, the exponent of a power of two.
//
// A power of two makes both directions exact but for the one rounding to a code: x / s and
// m s are exact in float32, and a code's value is exact in bfloat16.
#pragma once

#include "ltv_device.hpp"

namespace ltv {

constexpr int kFp4Block = 32;        // channels of a scale
constexpr int kFp4NaN = 255;         // a scale byte
constexpr int kFp4Low = 2, kFp4High = 252;

// Bytes of a token's head.
__host__ __device__ constexpr int fp4_row_bytes(int D) { return D / 2 + D / kFp4Block; }

// The scale's byte for a largest magnitude, given by its bits (NaN above infinity above all):
// of the smallest power of two of which it is at most 7.  (With 6 as the bound a block whose
// largest is between 6 and 7 would have all others half as exact to have that one no nearer:
// beside 7 the next larger scale has steps of 2.)  Monotone, so that the byte of a block is the
// largest of its parts'.
__device__ __forceinline__ int fp4_byte(uint32_t abs_bits) {
  const int e = (int)(abs_bits >> 23);
  const int byte = e - 2 + ((abs_bits & 0x7fffffu) > 0x600000u);
  return e == 255 ? kFp4NaN : min(max(byte, kFp4Low), kFp4High);
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The codes of eight values over s, of a byte that is not a NaN's: the conversion unit rounds to the
// nearest, ties to the even code, and takes 6 for what is beyond.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], int byte) {
  const float s = __uint_as_float((uint32_t)byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}

// x in float32, on the same side of all numbers of fewer bits, the borders of codes among them: what
// is between two float32 numbers becomes the one whose last bit is set, what is finite beyond them
// the largest (whose is).
__device__ __forceinline__ float beside(double x) {
  const float f = (float)x;
  if (fabsf(f) == INFINITY && fabs(x) < (double)INFINITY) return copysignf(3.4028234664e38f, f);
  const double d = x - (double)f;
  // (signs by their bits: f may be -0)
  const int bits = __float_as_int(f);
  const bool stay = d == 0.0 || (bits & 1) != 0 || !(fabsf(f) < INFINITY);
  return __int_as_float(bits + (stay ? 0 : (d < 0.0) == (bits < 0) ? 1 : -1));
}
// Two codes' values, of byte OF of a word, in bfloat16 (scale 2^(byte - 127), which all values
// are exact with; infinity, the scale byte of a NaN, makes NaNs).
template <int OF>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, OF));
}
__device__ __forceinline__ float scale_bits(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ uint4 fp4_eight(uint32_t codes, float s) {
  return make_uint4(fp4_pair<0>(codes, s), fp4_pair<1>(codes, s), fp4_pair<2>(codes, s),
                    fp4_pair<3>(codes, s));
}

}  // namespace ltv
