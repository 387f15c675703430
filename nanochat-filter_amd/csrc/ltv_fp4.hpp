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
__device__ __forceinline__ int fp4_byte(uint64_t abs_bits) {
  const int e = (int)(abs_bits >> 52);
  const int byte = e - 1023 + 127 - 2 + ((abs_bits & 0xfffffffffffffull) > 0xc000000000000ull);
  return e == 2047 ? kFp4NaN : min(max(byte, kFp4Low), kFp4High);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint64_t abs_bits(double x) {
  return (uint64_t)__double_as_longlong(x) & 0x7fffffffffffffffull;
}

// 1 / s of a byte
__device__ __forceinline__ float fp4_inverse(int byte, float) {
  return __uint_as_float((uint32_t)(254 - byte) << 23);
}
__device__ __forceinline__ double fp4_inverse(int byte, double) {
  return __longlong_as_double((long long)(1023 + 127 - byte) << 52);
}

// The code of x / s: the nearest, ties to the even one.
template <typename F>
__device__ __forceinline__ uint32_t fp4_code(F x, F inverse) {
  const F a = (x < 0 ? -x : x) * inverse;
  const uint32_t c = (a > (F)0.25) + (a >= (F)0.75) + (a > (F)1.25) + (a >= (F)1.75) +
                     (a > (F)2.5) + (a >= (F)3.5) + (a > (F)5.0);
  return c | (x < 0 ? 8u : 0u);
}

// s; a NaN for the byte of one.
__device__ __forceinline__ float fp4_scale(uint32_t byte) {
  return byte == kFp4NaN ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// The value of a code, without its scale.
__device__ __forceinline__ float fp4_value(uint32_t code) {
  const uint32_t m = code & 7;
  // 0.5 is the only one below 1; 1, 1.5, 2, 3, 4, 6 are 2^(m / 2 - 1) (1 + m % 2 / 2)
  const float f = m < 2 ? 0.5f * m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
  return code & 8 ? -f : f;
}

}  // namespace ltv
