// Attention of new tokens over a paged cache.
//
//   out[row] = sum_j p_j v_j,  p = softmax_{j <= pos(row)}(scale q[row] . k_j)
//
// One workgroup per (token, head): sixteen groups of sixteen lanes take the keys in
// turn, a lane holding eight of the head's channels; each group keeps a running
// maximum and sum, and the groups are joined at the end.
#include <algorithm>

#include "ltv_paged.hpp"

namespace ltv {
namespace {

struct AttnArgs {
  PagedBatch batch;
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  int64_t qs[3], ks[3], vs[3], os[3];  // elements
  int NH, NKVH, D;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnArgs a) {
  __shared__ float lds_ms[16][2];
  __shared__ float lds_o[16][128];
  const int h = blockIdx.y, b = blockIdx.z;
  const int kvh = h / (a.NH / a.NKVH);
  const PagedSeq s = paged_seq(a.batch, b);
  const int c = threadIdx.x & 15, gi = threadIdx.x >> 4;
  const bool on = c * 8 < a.D;
  for (int t = blockIdx.x; t < s.n; t += gridDim.x) {
    const int pos = s.len - s.n + t;
    const int64_t row = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;
    const int64_t qo = a.batch.starts != nullptr ? row * a.qs[1] : b * a.qs[0] + t * a.qs[1];
    const int64_t oo = a.batch.starts != nullptr ? row * a.os[1] : b * a.os[0] + t * a.os[1];
    const T* q = reinterpret_cast<const T*>(a.q) + qo + h * a.qs[2] + c * 8;
    float qf[8], o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[e] = on ? io_traits<T>::load(q + e) * a.scale : 0.0f;
      o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = gi; j <= pos; j += 16) {
      const int col = a.batch.div.quot(j);
      const int page = s.table[col];
      if (page < 0 || page >= a.batch.P) continue;
      const int at = j - col * a.batch.div.size;
      const T* k = reinterpret_cast<const T*>(a.k) + page * a.ks[0] + kvh * a.ks[1] +
                   at * a.ks[2] + c * 8;
      const T* v = reinterpret_cast<const T*>(a.v) + page * a.vs[0] + kvh * a.vs[1] +
                   at * a.vs[2] + c * 8;
      float x = 0.0f;
      if (on)
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf(qf[e], io_traits<T>::load(k + e), x);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
      const float mn = fmaxf(m, x);
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float was = __expf(m - base), p = __expf(x - base);
      l = l * was + p;
      m = mn;
      if (on)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(p, io_traits<T>::load(v + e), o[e] * was);
    }
    __syncthreads();
    if (c == 0) {
      lds_ms[gi][0] = m;
      lds_ms[gi][1] = l;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) lds_o[gi][c * 8 + e] = o[e];
    __syncthreads();
    float mx = -INFINITY;
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, lds_ms[i][0]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, acc = 0.0f;
    const int d = threadIdx.x;
    for (int i = 0; i < 16; ++i) {
      const float w = __expf(lds_ms[i][0] - base);
      sum = fmaf(lds_ms[i][1], w, sum);
      if (d < a.D) acc = fmaf(lds_o[i][d], w, acc);
    }
    if (d < a.D)
      io_traits<T>::store(reinterpret_cast<T*>(a.out) + oo + h * a.os[2] + d,
                          sum == 0.0f ? 0.0f : acc / sum);
    if (d == 0 && a.lse != nullptr)
      a.lse[row * a.NH + h] = sum == 0.0f ? -INFINITY : base + __logf(sum);
  }
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_paged_attention_workspace_size(int dtype, const ltv_paged_batch* batch,
                                                     int NH, int NKVH, int D, int max_len) {
  return 0;
}

extern "C" int ltv_paged_attention(int dtype, const void* q, const int64_t q_strides[3],
                                   const void* k_pages, const int64_t k_page_strides[3],
                                   const void* v_pages, const int64_t v_page_strides[3],
                                   const ltv_paged_batch* batch, void* out,
                                   const int64_t out_strides[3], float* lse, void* workspace,
                                   size_t workspace_bytes, int NH, int NKVH, int D, int max_len,
                                   float scale, void* stream) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  const int bad = check_batch(batch);
  if (bad != LTV_OK) return bad;
  LTV_REQUIRE(NH >= 0 && NKVH >= 0 && D > 0 && (NH == 0 || (NKVH > 0 && NH % NKVH == 0)),
              LTV_ERR_INVALID_ARG, "bad heads (NH=%d NKVH=%d D=%d)", NH, NKVH, D);
  LTV_REQUIRE(D % 8 == 0 && D <= 128, LTV_ERR_UNSUPPORTED,
              "head_dim must be a multiple of 8, at most 128 (D=%d)", D);
  if (batch->B == 0 || batch->total == 0 || NH == 0) return LTV_OK;
  LTV_REQUIRE(q && out && q_strides && out_strides && k_page_strides && v_page_strides &&
                  ((k_pages && v_pages) || batch->num_pages == 0),
              LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(scale > 0.0f && scale < INFINITY, LTV_ERR_INVALID_ARG,
              "scale must be positive and finite (%g)", scale);
  LTV_REQUIRE(batch->B <= 65535 && NH <= 65535, LTV_ERR_UNSUPPORTED,
              "more than 65,535 sequences or heads");
  AttnArgs a{PagedBatch(*batch), q, k_pages, v_pages, out, lse, {}, {}, {}, {}, NH, NKVH, D,
             scale};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.ks[i] = k_page_strides[i];
    a.vs[i] = v_page_strides[i];
    a.os[i] = out_strides[i];
  }
  const dim3 grid(std::max(1, std::min(batch->T, 65535)), NH, batch->B);
  if (dtype == LTV_DTYPE_F32)
    hipLaunchKernelGGL(attn_rows_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(attn_rows_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
