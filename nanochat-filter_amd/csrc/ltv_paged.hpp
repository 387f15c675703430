// What the kernels on the paged cache share: the sequences of a call as the device
// sees them, and host checks.  Every value that is read on the device (slots,
// starts, lengths, page ids) is brought into range here before it is an index.
#pragma once

#include "../../include/nanochat_serving_amd.h"
#include "ltv_abi_internal.hpp"
#include "ltv_device.hpp"

namespace ltv {

// n / size for 0 <= n < 2^31 by a multiplication: with l = ceil(log2 size) and
// m = floor(2^(31 + l) / size) + 1 the error of n m / 2^(31 + l) stays below 1 / size.
struct PageDiv {
  uint32_t mul;
  int shift;
  int size;
  explicit PageDiv(int s) : mul(0), shift(0), size(s) {
    int l = 0;
    while ((int64_t(1) << l) < s) ++l;
    if (l > 0) {
      mul = (uint32_t)(((uint64_t(1) << (31 + l)) / (uint64_t)s) + 1);
      shift = l - 1;
    }
  }
  __device__ __forceinline__ int quot(int n) const {
    return size == 1 ? n : quot_of_many(n);
  }
  __device__ __forceinline__ int quot_of_many(int n) const {  // (size > 1)
    return (int)(__umulhi((uint32_t)n, mul) >> shift);
  }
};

struct PagedBatch {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* slots;
  const int32_t* starts;
  int64_t table_stride, total;
  int B, T, S, P, W;
  PageDiv div;
  explicit PagedBatch(const ltv_paged_batch& b)
      : table(b.page_table), lens(b.seq_lens), slots(b.slots), starts(b.starts),
        table_stride(b.table_stride), total(b.total), B(b.B), T(b.T), S(b.num_slots),
        P(b.num_pages), W(b.table_width), div(b.page_size) {}
};

// Sequence b: its row of the table, tokens in the cache, new tokens and the row of the
// first of them (with starts) in the token tensors.
struct PagedSeq {
  const int32_t* table;
  int len, n;
  int64_t row0;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
  PagedSeq s;
  int slot = p.slots != nullptr ? p.slots[b] : b;
  const bool ok = slot >= 0 && slot < p.S;
  slot = ok ? slot : 0;
  s.table = p.table + (int64_t)slot * p.table_stride;
  const int64_t most = (int64_t)p.W * p.div.size;
  s.len = ok ? (int)min((int64_t)max(p.lens[slot], 0), min(most, (int64_t)0x7fffffff)) : 0;
  if (p.starts != nullptr) {
    const int64_t a = min((int64_t)max(p.starts[b], 0), p.total);
    const int64_t e = min((int64_t)max(p.starts[b + 1], 0), p.total);
    s.row0 = a;
    s.n = (int)max(e - a, (int64_t)0);
  } else {
    s.row0 = 0;
    s.n = p.T;
  }
  return s;
}

// Of a sequence: the kernels' positions run past its end by some tiles of keys, in 31 bits.
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 1024;

// Checks shared by the entry points that take a batch.
inline int check_batch(const ltv_paged_batch* b) {
  LTV_REQUIRE(b != nullptr, LTV_ERR_INVALID_ARG, "null batch");
  LTV_REQUIRE(b->B >= 0 && b->T >= 0 && b->num_slots >= 0 && b->num_pages >= 0 &&
                  b->table_width >= 0 && b->page_size > 0 && b->total >= 0 &&
                  b->table_stride >= b->table_width,
              LTV_ERR_INVALID_ARG,
              "bad batch (B=%d T=%d slots=%d pages=%d width=%d stride=%lld page size=%d)", b->B,
              b->T, b->num_slots, b->num_pages, b->table_width, (long long)b->table_stride,
              b->page_size);
  LTV_REQUIRE(b->page_size <= (1 << 20) &&
                  (int64_t)b->table_width * b->page_size <= kMostTokens &&
                  b->total < (int64_t(1) << 31),
              LTV_ERR_UNSUPPORTED, "a sequence's tokens and a call's new tokens must fit 31 bits");
  LTV_REQUIRE(b->starts != nullptr || b->total == (int64_t)b->B * b->T, LTV_ERR_INVALID_ARG,
              "without starts there are B * T token rows");
  LTV_REQUIRE(b->slots != nullptr || b->B <= b->num_slots, LTV_ERR_INVALID_ARG,
              "%d sequences, %d slots", b->B, b->num_slots);
  if (b->B > 0 && b->num_slots > 0)
    LTV_REQUIRE(b->seq_lens && (b->page_table || b->table_width == 0), LTV_ERR_INVALID_ARG,
                "null page table or lengths");
  return LTV_OK;
}

inline int elem_size(int dtype) { return dtype == LTV_DTYPE_F32 ? 4 : 2; }

}  // namespace ltv
