// What the pass over rows of logits leaves for other kernels to join: the pieces' sums and
// largest logits (ltv_logprobs.hip).
#pragma once

#include "../../include/nanochat_serving_amd.h"
#include "ltv_abi_internal.hpp"
#include "ltv_device.hpp"

namespace ltv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How z follows from x: none, by r, by tanh, by r in float64, by tanh in float64.
enum Cap { kNoCap, kCap, kWideCap, kCap64, kTanh64 };
constexpr float kMostCap = 64.0f;      // by r
constexpr float kMostCap64 = 0x1p20f;  // .. in float64

inline Cap cap_of(float softcap) {
  return softcap > kMostCap ? kWideCap : softcap > 0.0f ? kCap : kNoCap;
}

// .. where a float32 z of a large cap is too far off.
inline Cap exact_cap_of(float softcap) {
  const Cap c = cap_of(softcap);
  return c != kWideCap ? c : softcap <= kMostCap64 ? kCap64 : kTanh64;
}

// r of the cap's tanh; cap_scale = 2 log2(e) / c (finite for the smallest c, too)
__device__ __forceinline__ float cap_scale_of(float cap) {
  return fminf(2.0f * kLog2e / cap, 3.0e38f);
}
__device__ __forceinline__ float cap_r(float x, float cap_scale) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * cap_scale));
}
// c tanh(x / c) in float64: by 1 - tanh y = 2 / (e^{2 y} + 1), off by roundings of the cap (some
// 2^-32 at 2^20); of larger caps, beside which z may be small, to its own last bits, which takes
// twice as long (a pass over 384 rows of 50,257 bfloat16: 137 us, 62 so, and 22 with a cap of 15).
template <Cap CAP>
__device__ __forceinline__ double capped64(float x, double cap) {
  if constexpr (CAP == kNoCap) return x;
  const double y = (double)x / cap;
  return CAP != kTanh64 ? cap - 2.0 * cap / (exp(2.0 * y) + 1.0) : cap * tanh(y);
}
// e^z by r
__device__ __forceinline__ float cap_exp(float r, float cap) {
  const float at0 = cap * kLog2e, slope = -2.0f * at0;
  return __builtin_amdgcn_exp2f(fmaf(r, slope, at0));
}

// e^(z - m) as the pass has it
__device__ __forceinline__ float below_exp(double z, float m) {
  return __builtin_amdgcn_exp2f((float)(z - (double)m) * kLog2e);
}

// A total order of the logits with their indices: larger value first (NaN above all,
// -0 = +0), then lower index.  Never 0 for a real entry.
__device__ __forceinline__ uint64_t order_key(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  if (x != x) k = 0xffffffffu;
  return ((uint64_t)k << 32) | (uint32_t)(0x7fffffff - i);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ int key_index(uint64_t key) {
  return 0x7fffffff - (int)(uint32_t)key;
}

__device__ __forceinline__ uint64_t of_lane(uint64_t x, int i) {  // (i uniform)
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)x, i);
}

// The k-th largest of the 64 lanes' keys, 0 if fewer are not 0 (every lane gets it).
__device__ __forceinline__ uint64_t kth_of_lanes(uint64_t mine, int k) {
  int above = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) above += of_lane(mine, i) > mine;
  const uint64_t at = __ballot(above == k - 1 && mine != 0);
  return at == 0 ? 0 : of_lane(mine, __builtin_ctzll(at));
}

// Pieces that each of N rows of V logits is cut into.
int logprobs_pieces(int64_t N, int V);

// Of each piece of N <= 2^23 rows the sums (N, pieces, 3) -- m, S = sum e^(z - m) and one for
// the entropy; by r there is no m: S = sum e^z; of larger caps z is float64, and m its largest,
// a float32 number -- and the keys of its top_k largest logits (N, pieces, top_k), descending, 0
// where it has fewer.  Rows n with skip[n] are left out.
int logprobs_parts(int dtype, const void* x, int64_t row_stride, const uint8_t* skip,
                   float* part_sums, uint64_t* part_keys, int64_t N, int V, int top_k,
                   float softcap, hipStream_t stream);

}  // namespace ltv
