// New tokens on their way into the paged cache: queries and keys rotated by their
// positions and normalised, keys and values written into their pages as they are or in
// 4 bits; and the way back, what the pages hold of the new tokens.
//
//   y1 = x1 cos + x2 sin,  y2 = x2 cos - x1 sin   (x1, x2: the halves of a head)
//   y / sqrt(mean y^2 + eps)
//
// It is computed in float64 (bfloat16 results are rounded by way of float32, which moves one in
// 2^15 of them to the other side of a tie).  A code of 4 bits changes by up to half its size
// where a value crosses a border, so which side it is on is worth deciding right, and squares
// of large float32 values do not pass the range.
//
// Everything is read once and written once, in one launch for queries, keys and values.  Long
// prompts are bounded by the reads and by the float64 arithmetic about alike: 12,289 tokens of 12
// query and 4 k/v heads of 128, bfloat16 into 4-bit pages, 28 to 30 us (110 MB, 3.8 TB/s), and 9 us
// to read its keys and values back.  Small calls are latency, of the sequence's numbers, its page
// and its rows one after the other: 64 sequences of one token each 4.3 us, nine with chunks of up
// to 700 float32 tokens 7.1.
#include <algorithm>
#include <type_traits>

#include "../../include/nanochat_decoding_amd.h"
#include "ltv_fp4.hpp"
#include "ltv_paged.hpp"

namespace ltv {
namespace {

struct RotaryArgs {
  PagedBatch batch;
  const char* src[3];  // q, k, v
  int64_t ss[3][3];    // (sequence, token, head), bytes
  char* q_out;
  int64_t qo[3];
  char* pages[2];
  int64_t ps[2][3];  // (page, head, token), bytes
  const char* tab[2];
  int64_t ts[2];  // bytes from position to position
  int heads[3];
  int first;      // section of blockIdx.z == 0: 0, or 1 without queries
  int D, log_lanes;
  double eps;  // of the norm, negative: none
  double per_channel;  // 1 / D
  PageDiv by_heads[3];
};

// VEC elements at any alignment of the element.
template <typename T, int VEC>
__device__ __forceinline__ void load_floats(const char* p, float (&x)[VEC]) {
  T e[VEC];
  __builtin_memcpy(e, reinterpret_cast<const T*>(p), sizeof(e));
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = io_traits<T>::load(&e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_floats(char* p, const float (&x)[VEC]) {
  if constexpr (sizeof(T) == 4) {
    __builtin_memcpy(reinterpret_cast<float*>(p), x, sizeof(x));
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = cvt_pk_bf16(x[2 * i], x[2 * i + 1]);
    __builtin_memcpy(reinterpret_cast<bf16_t*>(p), w, sizeof(w));
  }
}

template <int CTRL>
__device__ __forceinline__ int quad_perm(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}

// Two chunks of eight channels of a token's head, half a head apart, into its 4-bit page: a lane of
// the row's `lanes` has chunks c and c + chunks.
__device__ __forceinline__ void store_fp4(const float (&y)[2][8], char* block, int in,
                                          int page_size, int D, int c, int chunks, int lanes) {
  int byte[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float top = fabsf(y[h][0]);  // (a NaN stays)
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_elementwise_maximum(top, fabsf(y[h][i]));
    byte[h] = fp4_byte(abs_bits(top));
  }
  // a scale's 32 channels are four chunks
  if ((chunks & 3) == 0) {  // .. of four lanes beside each other
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      byte[h] = max(byte[h], quad_perm<0xb1>(byte[h]));  // lanes 1, 0, 3, 2
      byte[h] = max(byte[h], quad_perm<0x4e>(byte[h]));  // lanes 2, 3, 0, 1
    }
  } else {  // .. of one half, or of both
    const int own = byte[0] | byte[1] << 8, lane0 = (threadIdx.x & 63) & ~(lanes - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = c + h * chunks;
      byte[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int other = (j & ~3) + i;
        const bool second = other >= chunks;
        const int theirs = __shfl(own, lane0 + (second ? other - chunks : other));
        byte[h] = max(byte[h], theirs >> (second ? 8 : 0) & 255);
      }
    }
  }
  if (c >= chunks) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = c + h * chunks;
    const bool nan = byte[h] == kFp4NaN;
    const uint32_t codes = fp4_codes(y[h], nan ? kFp4Low : byte[h]);
    *reinterpret_cast<uint32_t*>(block + in * (D / 2) + j * 4) = nan ? 0 : codes;
    if ((j & 3) == 0) block[page_size * (D / 2) + (j >> 2) * page_size + in] = (char)byte[h];
  }
}

// A group of lanes takes a token's head, a lane VEC channels of each half, so that a pair is in one
// lane and 16 bytes of bfloat16 (or four float32) one load; sums and scales go from lane to lane.
// Grid: (blocks over a sequence's tokens, B, q, k or v).  (Loading the next round's rows ahead, or
// four heads to a group of lanes that read the tables once, takes registers that the float64 values
// need: 12,289 tokens 39 to 52 us.)
template <typename T, typename TAB, int VEC, bool ROTATE, bool FP4>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  const int b = blockIdx.y, w = blockIdx.z + a.first;
  const PagedSeq s = paged_seq(a.batch, b);
  const int lanes = 1 << a.log_lanes, c = threadIdx.x & (lanes - 1);
  const int chunks = a.D / (2 * VEC), half = a.D / 2;
  const bool on = c < chunks;
  const int all = s.n * a.heads[w], step = (gridDim.x * 256) >> a.log_lanes;
  const int i0 = (blockIdx.x * 256 + threadIdx.x) >> a.log_lanes;
  // (all lanes of a wavefront go round together: they exchange sums and scales)
  const int rounds = (all + step - 1) / step;
  for (int round = 0; round < rounds; ++round) {
    const int i = i0 + round * step;
    const int t = a.by_heads[w].quot(min(i, all - 1)), h = min(i, all - 1) - t * a.heads[w];
    const int pos = s.len - s.n + t;
    const char* from = a.src[w] + (a.batch.starts != nullptr ? (s.row0 + t) * a.ss[w][1]
                                                             : b * a.ss[w][0] + t * a.ss[w][1]) +
                       h * a.ss[w][2];
    // (the row on its way before its page is looked up)
    float x[2][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[0][e] = x[1][e] = 0.0f;
    if (i < all && on) {
      load_floats<T, VEC>(from + c * VEC * sizeof(T), x[0]);
      load_floats<T, VEC>(from + (half + c * VEC) * sizeof(T), x[1]);
    }
    bool ok = i < all;
    int page = -1, in = 0;
    if (w > 0) {
      ok = ok && pos >= 0;
      if (ok) {
        const int col = a.batch.div.quot(pos);
        page = s.table[col];
        in = pos - col * a.batch.div.size;
        ok = page >= 0 && page < a.batch.P;
      }
    }
    [[maybe_unused]] double y[2][VEC];
    if constexpr (ROTATE) {
      if (w < 2) {
        if (ok && on && pos >= 0) {
          float cs[VEC], sn[VEC];
          load_floats<TAB, VEC>(a.tab[0] + pos * a.ts[0] + c * VEC * sizeof(TAB), cs);
          load_floats<TAB, VEC>(a.tab[1] + pos * a.ts[1] + c * VEC * sizeof(TAB), sn);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const double x1 = x[0][e], x2 = x[1][e], co = cs[e], si = sn[e];
            y[0][e] = fma(x1, co, x2 * si);
            y[1][e] = fma(x2, co, -(x1 * si));
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[0][e] = y[1][e] = 0.0;
        }
        if (a.eps >= 0.0) {
          double sum = 0.0;
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum = fma(y[0][e], y[0][e], fma(y[1][e], y[1][e], sum));
          for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor(sum, d);
          // (a token at a negative position stays 0, also with eps 0)
          const double r = pos < 0 ? 0.0 : rsqrt(fma(sum, a.per_channel, a.eps));
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            y[0][e] *= r;
            y[1][e] *= r;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[h][e] = FP4 && w == 1 ? beside(y[h][e]) : (float)y[h][e];
      }
    }
    if (FP4 && w > 0) {
      if constexpr (FP4) {
        // (no lane is left out: the scales are exchanged)
        const int at = ok ? page : 0;
        char* block = a.pages[w - 1] + at * a.ps[w - 1][0] + h * a.ps[w - 1][1];
        const int cc = ok ? c : chunks;  // (nothing is written)
        store_fp4(x, block, in, a.batch.div.size, a.D, cc, chunks, lanes);
      }
    } else if (ok && on) {
      char* to = w == 0 ? a.q_out + (a.batch.starts != nullptr ? (s.row0 + t) * a.qo[1]
                                                               : b * a.qo[0] + t * a.qo[1]) +
                              h * a.qo[2]
                        : a.pages[w - 1] + page * a.ps[w - 1][0] + h * a.ps[w - 1][1] +
                              in * a.ps[w - 1][2];
      store_floats<T, VEC>(to + c * VEC * sizeof(T), x[0]);
      store_floats<T, VEC>(to + (half + c * VEC) * sizeof(T), x[1]);
    }
  }
}

struct ReadArgs {
  PagedBatch batch;
  const char* pages[2];
  int64_t ps[2][3];  // (page, head, token), bytes
  char* out[2];
  int NKVH, D, units;  // units of a (token, head) row
  PageDiv by_row, by_units;
};

// One thread per unit of a token's row: eight channels (4 bits), or sizeof(U) bytes.  Grid: (blocks
// over a sequence's tokens, B and, with starts, one row more for the rows of no sequence, k or v).
template <typename U, typename T, bool FP4>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  constexpr int kOut = FP4 ? 8 * sizeof(T) : sizeof(U);  // bytes of a unit's output
  const int b = blockIdx.y, w = blockIdx.z;
  const unsigned per = (unsigned)a.NKVH * a.units, step = gridDim.x * 256;
  auto zero = [&](char* to) {
    if constexpr (FP4) {
#pragma unroll
      for (int e = 0; e < kOut; e += 16) *reinterpret_cast<uint4*>(to + e) = make_uint4(0, 0, 0, 0);
    } else {
      *reinterpret_cast<U*>(to) = U{};
    }
  };
  if (b == a.batch.B) {
    const int64_t first = min((int64_t)max(a.batch.starts[0], 0), a.batch.total);
    const int64_t last = min((int64_t)max(a.batch.starts[b], 0), a.batch.total);
    // (starts that do not ascend leave rows of no sequence between; they are written by none)
    const unsigned none = (unsigned)(a.batch.total - max(last - first, (int64_t)0)) * per;
    for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < none; i += step) {
      const unsigned before = (unsigned)first * per;
      zero(a.out[w] + (uint64_t)(i < before ? i : i - before + (unsigned)max(last, first) * per) * kOut);
    }
    return;
  }
  const PagedSeq s = paged_seq(a.batch, b);
  const unsigned all = (unsigned)s.n * per;  // (checked on the host)
  const int64_t row0 = a.batch.starts != nullptr ? s.row0 : (int64_t)b * a.batch.T;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const int t = a.by_row.quot((int)i), r = (int)i - t * (int)per;
    const int h = a.by_units.quot(r), u = r - h * a.units;
    char* to = a.out[w] + ((uint64_t)row0 * per + i) * kOut;
    const int pos = s.len - s.n + t;
    int page = -1, in = 0;
    if (pos >= 0) {
      const int col = a.batch.div.quot(pos);
      page = s.table[col];
      in = pos - col * a.batch.div.size;
    }
    if (page < 0 || page >= a.batch.P) {
      zero(to);
      continue;
    }
    const char* block = a.pages[w] + page * a.ps[w][0] + h * a.ps[w][1];
    if constexpr (FP4) {
      const int size = a.batch.div.size;
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(block + in * (a.D / 2) + u * 4);
      const uint4 x =
          fp4_eight(codes, scale_bits((uint8_t)block[size * (a.D / 2) + (u >> 2) * size + in]));
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(to) = x;
      } else {
        float f[8];
        unpack16(x, f, bf16_t());
        store_floats<T, 8>(to, f);
      }
    } else {
      *reinterpret_cast<U*>(to) = reinterpret_cast<const U*>(block + in * a.ps[w][2])[u];
    }
  }
}

int check_fp4(const ltv_paged_batch& b, const void* k_pages, const int64_t* ks,
              const void* v_pages, const int64_t* vs, int D) {
  LTV_REQUIRE(D % kFp4Block == 0 && D <= 128, LTV_ERR_UNSUPPORTED,
              "4-bit pages have head_dim 32, 64, 96 or 128 (D=%d)", D);
  LTV_REQUIRE(b.page_size % 16 == 0, LTV_ERR_UNSUPPORTED,
              "4-bit pages hold a multiple of 16 tokens (%d)", b.page_size);
  for (const int64_t* s : {ks, vs})
    LTV_REQUIRE(s[2] == fp4_row_bytes(D) && s[0] % 16 == 0 && s[1] % 16 == 0, LTV_ERR_UNSUPPORTED,
                "4-bit pages must be dense blocks, multiples of 16 bytes apart");
  LTV_REQUIRE(aligned16(k_pages) && aligned16(v_pages), LTV_ERR_UNSUPPORTED,
              "4-bit pages must be 16-byte aligned");
  return LTV_OK;
}

int check_call(int dtype, int page_format, const ltv_paged_batch* batch, int NH, int NKVH, int D) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  LTV_REQUIRE(page_format == LTV_PAGES_VALUES || page_format == LTV_PAGES_FP4,
              LTV_ERR_INVALID_ARG, "unknown page format %d", page_format);
  const int bad = check_batch(batch);
  if (bad != LTV_OK) return bad;
  LTV_REQUIRE(NH >= 0 && NKVH >= 0 && D > 0, LTV_ERR_INVALID_ARG,
              "bad heads (NH=%d NKVH=%d D=%d)", NH, NKVH, D);
  LTV_REQUIRE(D % 8 == 0 && D <= 128, LTV_ERR_UNSUPPORTED,
              "head_dim must be a multiple of 8, at most 128 (D=%d)", D);
  LTV_REQUIRE(batch->B <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 sequences in a call");
  LTV_REQUIRE(batch->total * std::max(NH, NKVH) < (int64_t(1) << 27), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  return LTV_OK;
}

template <typename T, typename TAB, int VEC, bool ROTATE, bool FP4>
void launch_rotary(const RotaryArgs& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((rotary_kernel<T, TAB, VEC, ROTATE, FP4>), grid, dim3(256), 0, st, a);
}

// Blocks over the new tokens of a sequence (T is a hint with starts: they stride over whatever
// there is).  Not more than twice what a sequence has on average, or most of them look and leave
// (chunks of nine sequences of up to 700 tokens 7.1 us, and 11 with blocks for the longest each),
// nor than go round a few times: each block's first round waits for its sequence's numbers, its
// page and its rows (12,289 tokens 28 us, with four times the blocks 45).
int blocks_for(const ltv_paged_batch& b, int64_t threads_per_token) {
  const int64_t longest = (std::max(b.T, 1) * threads_per_token + 255) / 256;
  const int64_t mean = (b.total * threads_per_token / std::max(b.B, 1) + 255) / 256;
  return (int)std::max<int64_t>(1, std::min({longest, 2 * mean, int64_t(1024)}));
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" int ltv_decoding_abi_version(void) { return 1; }

extern "C" int ltv_paged_rotary_append(
    int dtype, const void* q, const int64_t q_strides[3], const void* k,
    const int64_t k_strides[3], const void* v, const int64_t v_strides[3], const void* cos,
    int64_t cos_stride, const void* sin, int64_t sin_stride, int table_dtype, int64_t positions,
    double norm_eps, void* q_out, const int64_t q_out_strides[3], void* k_pages,
    const int64_t k_page_strides[3], void* v_pages, const int64_t v_page_strides[3],
    int page_format, const ltv_paged_batch* batch, int NH, int NKVH, int D, void* stream) {
  int bad = check_call(dtype, page_format, batch, NH, NKVH, D);
  if (bad != LTV_OK) return bad;
  LTV_REQUIRE(table_dtype == LTV_DTYPE_F32 || table_dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d of the tables", table_dtype);
  LTV_REQUIRE(norm_eps < (double)INFINITY, LTV_ERR_INVALID_ARG, "norm_eps must be finite");
  LTV_REQUIRE(positions >= (int64_t)batch->table_width * batch->page_size, LTV_ERR_INVALID_ARG,
              "tables of %lld positions, but the page table has room for %lld",
              (long long)positions, (long long)batch->table_width * batch->page_size);
  if (batch->B == 0 || batch->total == 0) return LTV_OK;
  // (nothing is kept of keys and values where there are no pages)
  const bool pages = NKVH > 0 && batch->num_pages > 0 && batch->num_slots > 0 &&
                     batch->table_width > 0;
  LTV_REQUIRE((NH == 0 || (q && q_strides && q_out && q_out_strides)) &&
                  (positions == 0 || (cos && sin)) &&
                  (!pages || (k && v && k_strides && v_strides && k_pages && v_pages &&
                              k_page_strides && v_page_strides)),
              LTV_ERR_INVALID_ARG, "null pointer");
  if (page_format == LTV_PAGES_FP4) {
    LTV_REQUIRE(D % kFp4Block == 0, LTV_ERR_UNSUPPORTED,
                "4-bit pages have head_dim 32, 64, 96 or 128 (D=%d)", D);
    if (pages) bad = check_fp4(*batch, k_pages, k_page_strides, v_pages, v_page_strides, D);
    if (bad != LTV_OK) return bad;
  }
  if (NH == 0 && !pages) return LTV_OK;
  const int es = elem_size(dtype), ts = elem_size(table_dtype);
  const bool fp4 = page_format == LTV_PAGES_FP4;
  const int vec = D % 16 == 0 && (dtype == LTV_DTYPE_BF16 || fp4) ? 8 : 4;
  int log_lanes = 0;
  while ((1 << log_lanes) < D / (2 * vec)) ++log_lanes;
  RotaryArgs a{PagedBatch(*batch), {(const char*)q, (const char*)k, (const char*)v}, {},
               (char*)q_out, {}, {(char*)k_pages, (char*)v_pages}, {},
               {(const char*)cos, (const char*)sin}, {cos_stride * ts, sin_stride * ts},
               {NH, NKVH, NKVH}, NH > 0 ? 0 : 1, D, log_lanes, norm_eps, 1.0 / D,
               {PageDiv(std::max(NH, 1)), PageDiv(std::max(NKVH, 1)), PageDiv(std::max(NKVH, 1))}};
  for (int i = 0; i < 3; ++i) {
    if (NH > 0) {
      a.ss[0][i] = q_strides[i] * es;
      a.qo[i] = q_out_strides[i] * es;
    }
    if (!pages) continue;
    a.ss[1][i] = k_strides[i] * es;
    a.ss[2][i] = v_strides[i] * es;
    a.ps[0][i] = k_page_strides[i] * (fp4 ? 1 : es);
    a.ps[1][i] = v_page_strides[i] * (fp4 ? 1 : es);
  }
  const int heads = std::max(NH, pages ? NKVH : 0);
  const dim3 grid(blocks_for(*batch, (int64_t)heads << log_lanes), batch->B,
                  (NH > 0) + (pages ? 2 : 0));
  const hipStream_t st = (hipStream_t)stream;
  auto by_table = [&](auto type, auto v, auto four) {
    using T = decltype(type);
    constexpr int V = decltype(v)::value;
    constexpr bool F = decltype(four)::value;
    if (table_dtype == LTV_DTYPE_F32) launch_rotary<T, float, V, true, F>(a, grid, st);
    else launch_rotary<T, bf16_t, V, true, F>(a, grid, st);
  };
  using V4 = std::integral_constant<int, 4>;
  using V8 = std::integral_constant<int, 8>;
  if (fp4) {
    if (dtype == LTV_DTYPE_F32) by_table(float(), V8(), std::true_type());
    else by_table(bf16_t(), V8(), std::true_type());
  } else if (dtype == LTV_DTYPE_F32) {
    by_table(float(), V4(), std::false_type());
  } else if (vec == 8) {
    by_table(bf16_t(), V8(), std::false_type());
  } else {
    by_table(bf16_t(), V4(), std::false_type());
  }
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" int ltv_paged_cache_append_fp4(int dtype, const void* k, const int64_t k_strides[3],
                                          const void* v, const int64_t v_strides[3], void* k_pages,
                                          const int64_t k_page_strides[3], void* v_pages,
                                          const int64_t v_page_strides[3],
                                          const ltv_paged_batch* batch, int NKVH, int D,
                                          void* stream) {
  int bad = check_call(dtype, LTV_PAGES_FP4, batch, 0, NKVH, D);
  if (bad != LTV_OK) return bad;
  if (batch->B == 0 || batch->total == 0 || NKVH == 0 || batch->num_pages == 0 ||
      batch->num_slots == 0 || batch->table_width == 0)
    return LTV_OK;
  LTV_REQUIRE(k && v && k_strides && v_strides && k_pages && v_pages && k_page_strides &&
                  v_page_strides,
              LTV_ERR_INVALID_ARG, "null pointer");
  bad = check_fp4(*batch, k_pages, k_page_strides, v_pages, v_page_strides, D);
  if (bad != LTV_OK) return bad;
  const int es = elem_size(dtype);
  int log_lanes = 0;
  while ((1 << log_lanes) < D / 16) ++log_lanes;
  RotaryArgs a{PagedBatch(*batch), {nullptr, (const char*)k, (const char*)v}, {}, nullptr, {},
               {(char*)k_pages, (char*)v_pages}, {}, {nullptr, nullptr}, {0, 0},
               {0, NKVH, NKVH}, 1, D, log_lanes, -1.0, 1.0 / D,
               {PageDiv(1), PageDiv(NKVH), PageDiv(NKVH)}};
  for (int i = 0; i < 3; ++i) {
    a.ss[1][i] = k_strides[i] * es;
    a.ss[2][i] = v_strides[i] * es;
    a.ps[0][i] = k_page_strides[i];
    a.ps[1][i] = v_page_strides[i];
  }
  const dim3 grid(blocks_for(*batch, (int64_t)NKVH << log_lanes), batch->B, 2);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == LTV_DTYPE_F32) launch_rotary<float, float, 8, false, true>(a, grid, st);
  else launch_rotary<bf16_t, float, 8, false, true>(a, grid, st);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" int ltv_paged_cache_read(int dtype, int page_format, const void* k_pages,
                                    const int64_t k_page_strides[3], const void* v_pages,
                                    const int64_t v_page_strides[3], const ltv_paged_batch* batch,
                                    void* k_out, void* v_out, int NKVH, int D, void* stream) {
  int bad = check_call(dtype, page_format, batch, 0, NKVH, D);
  if (bad != LTV_OK) return bad;
  if (batch->total == 0 || NKVH == 0) return LTV_OK;
  // (with starts there may be rows and no sequence)
  LTV_REQUIRE(batch->B > 0 || batch->starts != nullptr, LTV_ERR_INVALID_ARG,
              "rows of no sequence");
  LTV_REQUIRE(batch->B < 65535, LTV_ERR_UNSUPPORTED, "more than 65,534 sequences in a call");
  const bool pages = batch->num_pages > 0 && batch->num_slots > 0 && batch->table_width > 0;
  LTV_REQUIRE(k_out && v_out && (!pages || (k_pages && v_pages && k_page_strides && v_page_strides)),
              LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(aligned16(k_out) && aligned16(v_out), LTV_ERR_UNSUPPORTED,
              "the outputs must be 16-byte aligned");
  const bool fp4 = page_format == LTV_PAGES_FP4;
  if (fp4) {
    LTV_REQUIRE(D % kFp4Block == 0, LTV_ERR_UNSUPPORTED,
                "4-bit pages have head_dim 32, 64, 96 or 128 (D=%d)", D);
    if (pages) bad = check_fp4(*batch, k_pages, k_page_strides, v_pages, v_page_strides, D);
    if (bad != LTV_OK) return bad;
  }
  const int es = elem_size(dtype);
  ReadArgs a{PagedBatch(*batch), {(const char*)k_pages, (const char*)v_pages}, {},
             {(char*)k_out, (char*)v_out}, NKVH, D, 0, PageDiv(1), PageDiv(1)};
  uint64_t align = (uint64_t)k_pages | (uint64_t)v_pages | (uint64_t)(D * es);
  for (int i = 0; pages && i < 3; ++i) {
    a.ps[0][i] = k_page_strides[i] * (fp4 ? 1 : es);
    a.ps[1][i] = v_page_strides[i] * (fp4 ? 1 : es);
    align |= (uint64_t)a.ps[0][i] | (uint64_t)a.ps[1][i];
  }
  const bool wide = align % 16 == 0;
  a.units = fp4 ? D / 8 : wide ? D * es / 16 : D;
  LTV_REQUIRE(batch->total * NKVH * a.units < (int64_t(1) << 31), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  a.by_row = PageDiv(NKVH * a.units);
  a.by_units = PageDiv(a.units);
  const dim3 grid(blocks_for(*batch, (int64_t)NKVH * a.units),
                  batch->B + (batch->starts != nullptr ? 1 : 0), 2);
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto unit, auto type, auto four) {
    hipLaunchKernelGGL((read_kernel<decltype(unit), decltype(type), decltype(four)::value>), grid,
                       dim3(256), 0, st, a);
  };
  if (fp4) {
    if (dtype == LTV_DTYPE_F32) launch(0, float(), std::true_type());
    else launch(0, bf16_t(), std::true_type());
  } else if (wide) {
    launch(uint4(), float(), std::false_type());
  } else if (es == 4) {
    launch(uint32_t(), float(), std::false_type());
  } else {
    launch(uint16_t(), float(), std::false_type());
  }
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
