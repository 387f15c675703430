// Log probabilities of given tokens, entropy and top alternatives of rows of logits,
// and their gradient.
//
//   z = c tanh(x / c)  (or x),  m = max z,  S = sum e^{z - m},  A = sum (z - m) e^{z - m}
//   lse = m + log S,   logprob = z_t - lse,   entropy = log S - A / S
//
// One workgroup per row.
#include <algorithm>

#include "../../include/nanochat_serving_amd.h"
#include "ltv_abi_internal.hpp"
#include "ltv_device.hpp"

namespace ltv {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWaves = kRowThreads / 64;

struct LogpArgs {
  const void* x;
  int64_t xs;
  const int64_t* targets;
  float* logprobs;
  float* entropy;
  float* lse;
  float* top_lp;
  int64_t* top_ids;
  int V, top_k;
  float cap;
};

__device__ __forceinline__ float capped(float x, float cap) {
  return cap > 0.0f ? cap * tanhf(x / cap) : x;
}

// A total order of the logits with their indices: larger value first (NaN above all,
// -0 = +0), then lower index.  Never 0 for a real entry.
__device__ __forceinline__ uint64_t order_key(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  if (x != x) k = 0xffffffffu;
  return ((uint64_t)k << 32) | (uint32_t)(0x7fffffff - i);
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* lds, F f) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
  for (int w = 1; w < kRowWaves; ++w) r = f(r, lds[w]);
  return r;
}

__device__ __forceinline__ float f_add(float a, float b) { return a + b; }
// (NaN wins)
__device__ __forceinline__ float f_max(float a, float b) {
  return a != a ? a : b != b ? b : fmaxf(a, b);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprobs_forward_kernel(const LogpArgs a) {
  __shared__ float lds[kRowWaves];
  __shared__ unsigned long long best;
  const int64_t n = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.xs;
  const int tid = threadIdx.x;
  float m = -INFINITY;
  for (int j = tid; j < a.V; j += kRowThreads)
    m = f_max(m, capped(io_traits<T>::load(x + j), a.cap));
  m = block_reduce(m, lds, f_max);
  float s = 0.0f, t = 0.0f;
  for (int j = tid; j < a.V; j += kRowThreads) {
    const float d = capped(io_traits<T>::load(x + j), a.cap) - m, e = expf(d);
    s += e;
    if (!(e == 0.0f)) t = fmaf(d, e, t);
  }
  s = block_reduce(s, lds, f_add);
  t = block_reduce(t, lds, f_add);
  const float lse = m + logf(s);
  if (tid == 0) {
    const int64_t id = a.targets[n];
    a.logprobs[n] = id >= 0 && id < a.V
                        ? capped(io_traits<T>::load(x + id), a.cap) - lse : 0.0f;
    if (a.entropy != nullptr) a.entropy[n] = logf(s) - t / s;
    if (a.lse != nullptr) a.lse[n] = lse;
  }
  unsigned long long last = ~0ull;
  for (int i = 0; i < a.top_k; ++i) {
    unsigned long long mine = 0;
    for (int j = tid; j < a.V; j += kRowThreads) {
      const unsigned long long k = order_key(io_traits<T>::load(x + j), j);
      if (k < last && k > mine) mine = k;
    }
    __syncthreads();
    if (tid == 0) best = 0;
    __syncthreads();
    atomicMax(&best, mine);
    __syncthreads();
    last = best;
    const int j = 0x7fffffff - (int)(last & 0xffffffffu);
    if (tid == 0) {
      a.top_ids[n * a.top_k + i] = j;
      a.top_lp[n * a.top_k + i] = capped(io_traits<T>::load(x + j), a.cap) - lse;
    }
  }
}

struct LogpGradArgs {
  const void* x;
  int64_t xs;
  const int64_t* targets;
  const float* lse;
  const float* entropy;
  const int64_t* top_ids;
  const float* g_lp;
  const float* g_ent;
  const float* g_top;
  void* gx;
  int64_t gs;
  int V, top_k;
  float cap;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprobs_backward_kernel(const LogpGradArgs a) {
  const int64_t n = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.xs;
  T* gx = reinterpret_cast<T*>(a.gx) + n * a.gs;
  const int64_t target = a.targets[n];
  const bool given = target >= 0 && target < a.V;
  const float g = given && a.g_lp != nullptr ? a.g_lp[n] : 0.0f;
  const float ge = a.g_ent != nullptr ? a.g_ent[n] : 0.0f;
  const float ent = a.g_ent != nullptr ? a.entropy[n] : 0.0f;
  const int k = a.g_top != nullptr ? a.top_k : 0;
  float total = g;
  for (int i = 0; i < k; ++i) total += a.g_top[n * a.top_k + i];
  const float lse = a.lse[n];
  for (int j = threadIdx.x; j < a.V; j += kRowThreads) {
    const float z = capped(io_traits<T>::load(x + j), a.cap);
    const float lp = z - lse, p = expf(lp);
    float d = -p * total;
    if (!(p == 0.0f)) d -= ge * p * (lp + ent);
    if (j == target) d += g;
    for (int i = 0; i < k; ++i)
      if (a.top_ids[n * a.top_k + i] == j) d += a.g_top[n * a.top_k + i];
    if (a.cap > 0.0f) d *= 1.0f - (z / a.cap) * (z / a.cap);
    io_traits<T>::store(gx + j, d);
  }
}

int check_rows(int dtype, const void* x, int64_t row_stride, const int64_t* targets, int64_t N,
               int V, int top_k, float softcap) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  LTV_REQUIRE(N >= 0 && V > 0 && top_k >= 0 && top_k <= V, LTV_ERR_INVALID_ARG,
              "bad shape (N=%lld V=%d top_k=%d)", (long long)N, V, top_k);
  LTV_REQUIRE(top_k <= 64, LTV_ERR_UNSUPPORTED, "top_k is at most 64 (%d)", top_k);
  LTV_REQUIRE(softcap >= 0.0f && softcap < INFINITY, LTV_ERR_INVALID_ARG,
              "softcap must be finite and not negative");
  LTV_REQUIRE(N < (int64_t(1) << 31), LTV_ERR_UNSUPPORTED, "too many rows");
  if (N > 0) LTV_REQUIRE(x && targets, LTV_ERR_INVALID_ARG, "null pointer");
  return LTV_OK;
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" int ltv_token_logprobs_forward(int dtype, const void* logits, int64_t row_stride,
                                          const int64_t* targets, float* logprobs, float* entropy,
                                          float* lse, float* top_logprobs, int64_t* top_ids,
                                          int64_t N, int V, int top_k, float softcap,
                                          void* stream) {
  const int bad = check_rows(dtype, logits, row_stride, targets, N, V, top_k, softcap);
  if (bad != LTV_OK) return bad;
  if (N == 0) return LTV_OK;
  LTV_REQUIRE(logprobs && (top_k == 0 || (top_logprobs && top_ids)), LTV_ERR_INVALID_ARG,
              "null output");
  const LogpArgs a{logits, row_stride, targets, logprobs, entropy, lse, top_logprobs, top_ids,
                   V, top_k, softcap};
  if (dtype == LTV_DTYPE_F32)
    hipLaunchKernelGGL(logprobs_forward_kernel<float>, dim3((unsigned)N), dim3(kRowThreads), 0,
                       (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(logprobs_forward_kernel<bf16_t>, dim3((unsigned)N), dim3(kRowThreads), 0,
                       (hipStream_t)stream, a);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" int ltv_token_logprobs_backward(int dtype, const void* logits, int64_t row_stride,
                                           const int64_t* targets, const float* lse,
                                           const float* entropy, const int64_t* top_ids,
                                           const float* g_logprobs, const float* g_entropy,
                                           const float* g_top, void* grad_logits,
                                           int64_t grad_row_stride, int64_t N, int V, int top_k,
                                           float softcap, void* stream) {
  const int bad = check_rows(dtype, logits, row_stride, targets, N, V, top_k, softcap);
  if (bad != LTV_OK) return bad;
  if (N == 0) return LTV_OK;
  LTV_REQUIRE(lse && grad_logits && (!g_entropy || entropy) && (!g_top || top_k == 0 || top_ids),
              LTV_ERR_INVALID_ARG, "null pointer");
  const LogpGradArgs a{logits, row_stride, targets, lse, entropy, top_ids, g_logprobs, g_entropy,
                       g_top, grad_logits, grad_row_stride, V, top_k, softcap};
  if (dtype == LTV_DTYPE_F32)
    hipLaunchKernelGGL(logprobs_backward_kernel<float>, dim3((unsigned)N), dim3(kRowThreads), 0,
                       (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(logprobs_backward_kernel<bf16_t>, dim3((unsigned)N), dim3(kRowThreads), 0,
                       (hipStream_t)stream, a);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
