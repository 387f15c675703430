// Attention of new tokens over a paged cache held in 4 bits.
//
//   out[row] = sum_j p_j v_j,  p = softmax_{j <= pos(row)}(scale q[row] . k_j)
//
// k and v are the values that the codes and scales stand for.
#include "../../include/nanochat_decoding_amd.h"
#include "ltv_fp4.hpp"
#include "ltv_paged_line.hpp"

namespace ltv {
namespace {

// Keys and values of 4-bit pages, for rows_one_by_one.
struct Fp4Pages {
  static __device__ __forceinline__ void load(const char* block, const AttnArgs& a, uint32_t in,
                                              int c, float (&x)[8]) {
    const int size = a.batch.div.size;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(block + in * (a.D / 2) + c * 4);
    const float s = fp4_scale((uint8_t)block[size * (a.D / 2) + (c >> 2) * size + in]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fp4_value(codes >> (4 * e) & 15) * s;
  }
  static __device__ __forceinline__ void keys(const AttnArgs& a, int kvh, int page, uint32_t in,
                                              int c, float (&x)[8]) {
    load(a.k + kvh * a.kh + (uint64_t)((uint32_t)page * (uint64_t)a.kp) * 16, a, in, c, x);
  }
  static __device__ __forceinline__ void values(const AttnArgs& a, int kvh, int page, uint32_t in,
                                                int c, float (&x)[8]) {
    load(a.v + kvh * a.vh + (uint64_t)((uint32_t)page * (uint64_t)a.vp) * 16, a, in, c, x);
  }
};

constexpr int kRowsEach = 16;  // of a workgroup

template <typename T>
__global__ void __launch_bounds__(256) attn4_rows_kernel(const AttnArgs a) {
  __shared__ float lds[16 * 130];
  const int b = blockIdx.z, kvh = blockIdx.y;
  const PagedSeq s = paged_seq(a.batch, b);
  const int rows = s.n * a.g;
  for (int row0 = blockIdx.x * kRowsEach; row0 < rows; row0 += gridDim.x * kRowsEach) {
    const int end = min(rows, row0 + kRowsEach);
    const int keys = max(s.len - s.n + a.by_g.quot(end - 1) + 1, 0);
    rows_one_by_one<T, 256, Fp4Pages>(a, s, b, kvh, row0, end, 0, keys, -1, lds);
  }
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_paged_attention_fp4_workspace_size(int dtype, const ltv_paged_batch* batch,
                                                         int NH, int NKVH, int D, int max_len) {
  return 0;
}

extern "C" int ltv_paged_attention_fp4(int dtype, const void* q, const int64_t q_strides[3],
                                       const void* k_pages, const int64_t k_page_strides[3],
                                       const void* v_pages, const int64_t v_page_strides[3],
                                       const ltv_paged_batch* batch, void* out,
                                       const int64_t out_strides[3], float* lse, void* workspace,
                                       size_t workspace_bytes, int NH, int NKVH, int D,
                                       int max_len, float scale, void* stream) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  const int bad = check_batch(batch);
  if (bad != LTV_OK) return bad;
  LTV_REQUIRE(NH >= 0 && NKVH >= 0 && D > 0 && (NH == 0 || (NKVH > 0 && NH % NKVH == 0)),
              LTV_ERR_INVALID_ARG, "bad heads (NH=%d NKVH=%d D=%d)", NH, NKVH, D);
  LTV_REQUIRE(D % kFp4Block == 0 && D <= 128, LTV_ERR_UNSUPPORTED,
              "4-bit pages have head_dim 32, 64, 96 or 128 (D=%d)", D);
  LTV_REQUIRE(batch->page_size % 16 == 0, LTV_ERR_UNSUPPORTED,
              "4-bit pages hold a multiple of 16 tokens (%d)", batch->page_size);
  LTV_REQUIRE(scale > 0.0f && scale * kLog2e < INFINITY, LTV_ERR_INVALID_ARG,
              "scale must be positive and finite (%g)", scale);
  if (batch->B == 0 || batch->total == 0 || NH == 0) return LTV_OK;
  LTV_REQUIRE(batch->total * NH < (int64_t(1) << 30), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  LTV_REQUIRE(batch->B <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 sequences in a call");
  const bool pages = batch->num_pages > 0;
  LTV_REQUIRE(q && out && q_strides && out_strides &&
                  (!pages || (k_pages && v_pages && k_page_strides && v_page_strides)),
              LTV_ERR_INVALID_ARG, "null pointer");
  if (pages) {
    for (const int64_t* s : {k_page_strides, v_page_strides}) {
      LTV_REQUIRE(s[2] == fp4_row_bytes(D) && s[0] % 16 == 0 && s[1] % 16 == 0,
                  LTV_ERR_UNSUPPORTED,
                  "4-bit pages must be dense blocks, multiples of 16 bytes apart");
      LTV_REQUIRE(s[0] >= 0 && s[1] >= 0 &&
                      (s[0] == 0 || batch->num_pages <= (int64_t(1) << 35) / s[0]),
                  LTV_ERR_UNSUPPORTED,
                  "the pages of a layer must lie within 32 GiB, with strides that are not negative");
    }
    LTV_REQUIRE(aligned16(k_pages) && aligned16(v_pages), LTV_ERR_UNSUPPORTED,
                "4-bit pages must be 16-byte aligned");
  }
  const int es = elem_size(dtype);
  AttnArgs a{PagedBatch(*batch), (const char*)q, (const char*)k_pages, (const char*)v_pages,
             (char*)out, lse, (float*)workspace, {}, {},
             pages ? k_page_strides[1] : 0, pages ? v_page_strides[1] : 0,
             pages ? (uint32_t)(k_page_strides[0] / 16) : 0, 0,
             pages ? (uint32_t)(v_page_strides[0] / 16) : 0, 0, NH, NKVH, D, NH / NKVH, 0, 1, 0,
             scale * kLog2e, 0, 0, 0, 0, 0, 0, 0, 0, 0, PageDiv(NH / NKVH), PageDiv(1), 0,
             nullptr, nullptr};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i] * es;
    a.os[i] = out_strides[i] * es;
  }
  const int64_t rows = (int64_t)std::max(batch->T, 1) * (NH / NKVH);
  const dim3 grid((unsigned)std::min<int64_t>((rows + kRowsEach - 1) / kRowsEach, 1024), NKVH,
                  batch->B);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == LTV_DTYPE_F32)
    hipLaunchKernelGGL(attn4_rows_kernel<float>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(attn4_rows_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
