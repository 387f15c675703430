// The paged cache: writing new tokens into their pages, and the pages' bookkeeping --
// reserve (with copies of shared pages), fork, free, copy, compact -- on the device,
// so that a serving loop needs no host copy of the page table and no wait.
//
// All of it is integer work and copies.  The bookkeeping is small (one workgroup
// scans the reference counts; 64 Ki pages are 256 KB) and bounded by latency; the
// copies are bounded by HBM: each byte read once, written once.
#include <algorithm>

#include "../../include/nanochat_decoding_amd.h"
#include "ltv_paged.hpp"

namespace ltv {
namespace {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
  PagedBatch batch;
  const char* src[2];
  char* pages[2];
  int64_t ss[2][3];  // (sequence, token, head), bytes
  int64_t ps[2][3];  // (page, head, token), bytes
  int NKVH, units;   // units of kUnit bytes per (token, head) row
};

// One thread per unit (16 bytes, or one element where the rows are not aligned) of a
// token's rows of one tensor.  Grid: (blocks over a sequence's tokens, B, k or v).  Bounded
// by memory for chunks (12,289 tokens of 6 heads of 128, 75 MB read and written, 14 us: 5.4
// TB/s) and by the way to a page, three loads one after the other, for single tokens (3 us).
template <typename U>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  const int b = blockIdx.y, w = blockIdx.z;
  const PagedSeq s = paged_seq(a.batch, b);
  const int per = a.NKVH * a.units;  // units of one token
  const unsigned all = (unsigned)s.n * (unsigned)per;  // (checked on the host)
  const unsigned step = gridDim.x * 256;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const int t = (int)(i / (unsigned)per), r = (int)(i - (unsigned)t * per);
    const int h = r / a.units, u = r - h * a.units;
    const int pos = s.len - s.n + t;
    if (pos < 0) continue;
    const int col = a.batch.div.quot(pos);
    const int page = s.table[col];
    if (page < 0 || page >= a.batch.P) continue;
    const char* from = a.src[w] + (a.batch.starts != nullptr ? (s.row0 + t) * a.ss[w][1]
                                                             : b * a.ss[w][0] + t * a.ss[w][1]) +
                       h * a.ss[w][2];
    char* to = a.pages[w] + page * a.ps[w][0] + h * a.ps[w][1] +
               (pos - col * a.batch.div.size) * a.ps[w][2];
    reinterpret_cast<U*>(to)[u] = reinterpret_cast<const U*>(from)[u];
  }
}

// ---------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------
struct CopyArgs {
  char* base[2];
  int64_t page_b[2], layer_b[2];
  int64_t units;  // 16-byte units of a page block
  int layers, P;
};

inline CopyArgs copy_args(const ltv_page_blocks& b) {
  CopyArgs c;
  c.base[0] = reinterpret_cast<char*>(b.k);
  c.base[1] = reinterpret_cast<char*>(b.v);
  c.page_b[0] = b.k_page_bytes;
  c.page_b[1] = b.v_page_bytes;
  c.layer_b[0] = b.k_layer_bytes;
  c.layer_b[1] = b.v_layer_bytes;
  c.units = b.block_bytes / 16;
  c.layers = b.layers;
  c.P = b.num_pages;
  return c;
}

constexpr int kCopyThreads = 256;
constexpr int kCopyUnits = 2;                            // 16-byte units per thread
constexpr int kCopyPiece = kCopyThreads * kCopyUnits;    // units per workgroup step
constexpr int kCopyGrid = 2048;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Copies pages src[i] -> dst[i], i < count, over all layers and both tensors: the work
// is cut into pieces of 8 KiB which the workgroups take in turn.  Measured: 8 pages of 12
// layers (38 MB read and written) 5.2 us, 192 of them 184 us (4.9 TB/s, what a large copy
// reaches); stores that stay in the caches 6.1 and 188 us; pieces of 16 KiB 5.5 and 186 us.
// The indices are of 32 bits: divisions of 64 took 14 us of the small copy.
__device__ __forceinline__ void copy_pages(const CopyArgs& c, const int32_t* src,
                                           const int32_t* dst, int count) {
  const unsigned per_block = (unsigned)((c.units + kCopyPiece - 1) / kCopyPiece);
  const unsigned pieces = (unsigned)count * c.layers * 2 * per_block;  // (checked on the host)
  for (unsigned i = blockIdx.x; i < pieces; i += gridDim.x) {
    const unsigned j = i / per_block;
    const int at = (int)(i - j * per_block) * kCopyPiece;
    const int w = (int)(j & 1);
    const unsigned pl = j >> 1;
    const unsigned p = pl / (unsigned)c.layers;
    const int layer = (int)(pl - p * c.layers);
    const int from = src[p], to = dst[p];
    if (from < 0 || to < 0 || from >= c.P || to >= c.P || from == to) continue;
    char* base = c.base[w] + layer * c.layer_b[w];
    const u32x4* f = reinterpret_cast<const u32x4*>(base + from * c.page_b[w]);
    u32x4* t = reinterpret_cast<u32x4*>(base + to * c.page_b[w]);
    u32x4 x[kCopyUnits];
#pragma unroll
    for (int e = 0; e < kCopyUnits; ++e) {
      const int u = at + e * kCopyThreads + threadIdx.x;
      if (u < c.units) x[e] = f[u];
    }
#pragma unroll
    for (int e = 0; e < kCopyUnits; ++e) {
      const int u = at + e * kCopyThreads + threadIdx.x;
      if (u < c.units) __builtin_nontemporal_store(x[e], t + u);
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const CopyArgs c, const int32_t* src,
                                                            const int32_t* dst,
                                                            const int32_t* count, int n) {
  copy_pages(c, src, dst, count != nullptr ? min(*count, n) : n);
}

// ---------------------------------------------------------------------------
// bookkeeping
// ---------------------------------------------------------------------------
struct State {
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  int64_t ts;
  int S, W, P, page;
};

inline State state_of(const ltv_page_state& s) {
  return State{s.page_table, s.seq_lens, s.ref_counts, s.table_stride, s.num_slots,
               s.table_width, s.num_pages, s.page_size};
}

__device__ __forceinline__ bool in(int i, int n) { return i >= 0 && i < n; }
// Pages of `len` tokens (len + page - 1 may pass 31 bits, not 32).
__device__ __forceinline__ int pages_of(int len, int page) {
  return (int)(((unsigned)len + (unsigned)page - 1) / (unsigned)page);
}

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / 64;

// Exclusive sum of v over the workgroup's threads, and the total.
template <typename N>
__device__ __forceinline__ N block_scan(N v, N* lds, N& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  N x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const N y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // (lds may still be read from the scan before)
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  N before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kScanWaves; ++w) {
    const N t = lds[w];
    before += w < wave ? t : 0;
    total += t;
  }
  return before + x - v;
}

struct ReserveWs {
  int32_t* first;   // (n) first new page's rank among the free pages
  int32_t* plan;    // (n) 1: copy the last page; -1: nothing to do
  int32_t* writers; // (P) slots of this call that write into the page
  int32_t* last;    // (P) the last of them
  int32_t* src;     // (n) pages to copy
  int32_t* dst;
  int32_t* count;   // copies
};

inline size_t reserve_ws_ints(int n, int P) { return 4 * (size_t)n + 2 * (size_t)P + 1; }

// One workgroup.  What an entry needs follows from the state before the call and from
// the other entries that hold its last page, so the entries are planned in parallel:
// first the writers of each partly filled page are counted, then a scan over the
// entries' needs gives each its rank among the free pages, then a scan over the
// reference counts hands the free pages out.  All latency: 8 entries and 70 pages 7.8 us, 192
// entries and 900 pages 10.4.  (Entries kept in registers and LDS, the counts read ahead: 7.1
// and 13.5.)
//
// N: what the pages wanted are counted in, 64 bits where n rows of W pages pass 31 (192 entries
// 10.8 us with them, 10.2 without).
template <typename N>
__global__ void __launch_bounds__(kScanThreads) reserve_kernel(const State s,
                                                               const int32_t* slots,
                                                               const int32_t* counts, int n,
                                                               const ReserveWs ws,
                                                               int32_t* status) {
  __shared__ int lds[kScanWaves];
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0;
  __syncthreads();

  // an entry's slot and lengths, and the page that its new tokens begin in, if that is
  // partly filled; false: out of range
  auto read_entry = [&](int i, int& slot, int& old, int& len, int& last) {
    slot = slots[i];
    const int c = counts[i];
    if (!in(slot, s.S) || c < 0) return false;
    old = s.lens[slot];
    if (old < 0 || (int64_t)old + c > (int64_t)s.W * s.page) return false;
    len = old + c;
    last = -1;
    if (c > 0 && old % s.page != 0) last = s.table[slot * s.ts + old / s.page];
    return true;
  };
  // (a thread's first entry is read once)
  int slot0 = 0, old0 = 0, len0 = 0, last0 = -1;
  const bool ok0 = tid < n && read_entry(tid, slot0, old0, len0, last0);
  auto entry = [&](int i, int& slot, int& old, int& len, int& last) {
    if (i != tid) return read_entry(i, slot, old, len, last);
    slot = slot0;
    old = old0;
    len = len0;
    last = last0;
    return ok0;
  };

  for (int i = tid; i < n; i += kScanThreads) {
    int slot, old, len, last;
    if (!entry(i, slot, old, len, last)) {
      bad = 1;
    } else if (in(last, s.P)) {
      ws.writers[last] = 0;
      ws.last[last] = -1;
    }
  }
  __syncthreads();
  if (bad) {
    if (tid == 0) {
      *status = -1;
      *ws.count = 0;
    }
    return;
  }
  for (int i = tid; i < n; i += kScanThreads) {
    int slot, old, len, last;
    entry(i, slot, old, len, last);
    if (in(last, s.P)) {
      atomicAdd(&ws.writers[last], 1);
      atomicMax(&ws.last[last], i);
    }
  }
  __threadfence_block();
  __syncthreads();
  __shared__ N needs[kScanWaves];
  N wanted = 0;  // (uniform)
  for (int i0 = 0; i0 < n; i0 += kScanThreads) {
    const int i = i0 + tid;
    int need = 0, copy = 0;
    if (i < n) {
      int slot, old, len, last;
      entry(i, slot, old, len, last);
      if (in(last, s.P)) {
        const int r = s.refs[last];
        const int w = __hip_atomic_load(&ws.writers[last], __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
        const int l = __hip_atomic_load(&ws.last[last], __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
        copy = r > w || (r > 1 && l != i);
      }
      need = copy + pages_of(len, s.page) - pages_of(old, s.page);
    }
    N total;
    const N before = block_scan((N)need, needs, total);
    if (i < n) {
      ws.first[i] = (int)(wanted + before);  // (read where there are enough)
      ws.plan[i] = copy;
    }
    wanted += total;
  }
  // enough free pages?
  int free_pages = 0;
  for (int p0 = 0; p0 < s.P && free_pages < wanted; p0 += kScanThreads) {
    const int p = p0 + tid;
    int total;
    block_scan((int)(p < s.P && s.refs[p] == 0), lds, total);
    free_pages += total;
  }
  if (free_pages < wanted) {
    if (tid == 0) {
      *status = (int)min(wanted - (N)free_pages, (N)0x7fffffff);
      *ws.count = 0;
    }
    return;
  }
  __syncthreads();
  // hand them out: the free page of rank r goes to the last entry whose first rank is
  // <= r and which needs a page
  int rank0 = 0;
  for (int p0 = 0; p0 < s.P && rank0 < wanted; p0 += kScanThreads) {
    const int p = p0 + tid;
    const bool is_free = p < s.P && s.refs[p] == 0;
    int total;
    const int rank = rank0 + block_scan((int)is_free, lds, total);
    if (is_free && rank < wanted) {
      int lo = 0, hi = n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ws.first[mid] <= rank) lo = mid; else hi = mid - 1;
      }
      int slot, old, len, last;
      entry(lo, slot, old, len, last);
      const int j = rank - ws.first[lo];
      const int copy = ws.plan[lo];
      int32_t* row = s.table + slot * s.ts;
      if (copy && j == 0) {
        ws.src[lo] = last;
        ws.dst[lo] = p;
      } else {
        row[pages_of(old, s.page) + j - copy] = p;
      }
      s.refs[p] = 1;
    }
    rank0 += total;
  }
  __syncthreads();
  // lengths, the copied pages' places, and the list of copies
  int copies = 0;
  for (int i0 = 0; i0 < n; i0 += kScanThreads) {
    const int i = i0 + tid;
    int copy = 0, from = 0, to = 0;
    if (i < n) {
      int slot, old, len, last;
      // (a slot named twice may have grown meanwhile: checked again)
      if (entry(i, slot, old, len, last)) {
        copy = ws.plan[i];
        if (copy) {
          from = ws.src[i];
          to = ws.dst[i];
          s.table[slot * s.ts + old / s.page] = to;
          atomicSub(&s.refs[from], 1);
        }
        s.lens[slot] = len;
      }
    }
    int total;
    const int at = copies + block_scan(copy, lds, total);  // (at <= i: read before it is written)
    if (copy) {
      ws.src[at] = from;
      ws.dst[at] = to;
    }
    copies += total;
  }
  if (tid == 0) {
    *status = 0;
    *ws.count = copies;
  }
}

__global__ void __launch_bounds__(256) fork_kernel(const State s, const int32_t* src,
                                                   const int32_t* dst) {
  const int i = blockIdx.y, from = src[i], to = dst[i];
  if (!in(from, s.S) || !in(to, s.S) || from == to) return;
  for (int c = blockIdx.x * 256 + threadIdx.x; c < s.W; c += gridDim.x * 256) {
    int32_t* at = s.table + to * s.ts + c;
    const int page = s.table[from * s.ts + c], old = *at;
    if (in(page, s.P)) atomicAdd(&s.refs[page], 1);
    if (in(old, s.P)) atomicSub(&s.refs[old], 1);
    *at = page;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) s.lens[to] = s.lens[from];
}

// Reordering: what is wanted of a column is read, and the counts follow, before any of it is
// written.  The columns do not meet: a workgroup takes some of them, for all entries at once, in
// LDS.  All latency: 4 entries of 10 pages 1.8 us, 384 of 502 pages (1.5 MB of table) 5.6.
constexpr int kReorderInts = 8192, kReorderThreads = 1024;

__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const State s,
                                                                  const int32_t* slots,
                                                                  const int32_t* src, int n,
                                                                  int log_cols) {
  __shared__ int rows[kReorderInts];
  __shared__ int lens[kReorderInts >> 2];  // (four columns at least)
  const int c0 = blockIdx.x << log_cols, mask = (1 << log_cols) - 1;
  for (int u = threadIdx.x; u < n << log_cols; u += kReorderThreads) {
    const int i = u >> log_cols, c = c0 + (u & mask), from = src[i], to = slots[i];
    if (!in(from, s.S) || !in(to, s.S)) continue;
    if (blockIdx.x == 0 && (u & mask) == 0) lens[i] = s.lens[from];
    if (c >= s.W) continue;
    const int page = s.table[from * s.ts + c], old = s.table[to * s.ts + c];
    if (page != old) {
      if (in(page, s.P)) atomicAdd(&s.refs[page], 1);
      if (in(old, s.P)) atomicSub(&s.refs[old], 1);
    }
    rows[u] = page;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < n << log_cols; u += kReorderThreads) {
    const int i = u >> log_cols, c = c0 + (u & mask), from = src[i], to = slots[i];
    if (!in(from, s.S) || !in(to, s.S)) continue;
    if (blockIdx.x == 0 && (u & mask) == 0) s.lens[to] = lens[i];
    if (c < s.W) s.table[to * s.ts + c] = rows[u];
  }
}

// Of more entries than that, by way of memory.
__global__ void __launch_bounds__(256) reorder_read_kernel(const State s, const int32_t* slots,
                                                           const int32_t* src, int32_t* rows,
                                                           int32_t* lens) {
  const int i = blockIdx.y, from = src[i], to = slots[i];
  if (!in(from, s.S) || !in(to, s.S)) return;
  for (int c = blockIdx.x * 256 + threadIdx.x; c < s.W; c += gridDim.x * 256) {
    const int page = s.table[from * s.ts + c], old = s.table[to * s.ts + c];
    if (page != old) {
      if (in(page, s.P)) atomicAdd(&s.refs[page], 1);
      if (in(old, s.P)) atomicSub(&s.refs[old], 1);
    }
    rows[(int64_t)i * s.W + c] = page;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) lens[i] = s.lens[from];
}

__global__ void __launch_bounds__(256) reorder_write_kernel(const State s, const int32_t* slots,
                                                            const int32_t* src,
                                                            const int32_t* rows,
                                                            const int32_t* lens) {
  const int i = blockIdx.y, from = src[i], to = slots[i];
  if (!in(from, s.S) || !in(to, s.S)) return;
  for (int c = blockIdx.x * 256 + threadIdx.x; c < s.W; c += gridDim.x * 256)
    s.table[to * s.ts + c] = rows[(int64_t)i * s.W + c];
  if (blockIdx.x == 0 && threadIdx.x == 0) s.lens[to] = lens[i];
}

__global__ void __launch_bounds__(256) free_kernel(const State s, const int32_t* slots) {
  const int slot = slots[blockIdx.y];
  if (!in(slot, s.S)) return;
  for (int c = blockIdx.x * 256 + threadIdx.x; c < s.W; c += gridDim.x * 256) {
    // (an exchange: a slot named twice lets its pages go once)
    const int page = atomicExch(&s.table[slot * s.ts + c], -1);
    if (in(page, s.P)) atomicSub(&s.refs[page], 1);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) s.lens[slot] = 0;
}

struct CompactWs {
  int32_t* place;   // (P) where each page goes
  int32_t* movers;  // (P)
  int32_t* holes;   // (P)
  int32_t* count;
};

inline size_t compact_ws_ints(int P) { return 3 * (size_t)P + 1; }

// One workgroup: the pages in use are counted, then those past the count and the holes
// before it are listed in order; as many of one as of the other.
__global__ void __launch_bounds__(kScanThreads) compact_plan_kernel(const State s,
                                                                    const CompactWs ws,
                                                                    int32_t* live) {
  __shared__ int lds[kScanWaves];
  const int tid = threadIdx.x;
  int used = 0;
  for (int p = tid; p < s.P; p += kScanThreads) used += s.refs[p] > 0;
  int L;
  block_scan(used, lds, L);
  int movers = 0, holes = 0;
  for (int p0 = 0; p0 < s.P; p0 += kScanThreads) {
    const int p = p0 + tid;
    const bool use = p < s.P && s.refs[p] > 0;
    const bool mover = use && p >= L, hole = p < s.P && !use && p < L;
    // (both kinds in one scan: movers in the high half, at most 1,024 each)
    int total;
    const int before = block_scan((mover << 16) + hole, lds, total);
    if (mover) ws.movers[movers + (before >> 16)] = p;
    if (hole) ws.holes[holes + (before & 0xffff)] = p;
    if (p < s.P) ws.place[p] = p;
    movers += total >> 16;
    holes += total & 0xffff;
  }
  __syncthreads();
  for (int i = tid; i < movers; i += kScanThreads) {
    const int from = ws.movers[i], to = ws.holes[i];
    ws.place[from] = to;
    s.refs[to] = s.refs[from];
    s.refs[from] = 0;
  }
  if (tid == 0) {
    *ws.count = movers;
    *live = L;
  }
}

__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(const CopyArgs c,
                                                                    const State s,
                                                                    const CompactWs ws) {
  const int count = *ws.count;
  if (count == 0) return;
  for (int slot = blockIdx.x; slot < s.S; slot += gridDim.x)
    for (int col = threadIdx.x; col < s.W; col += kCopyThreads) {
      int32_t* at = s.table + slot * s.ts + col;
      const int page = *at;
      if (in(page, s.P)) {
        const int to = ws.place[page];
        if (to != page) *at = to;
      }
    }
  copy_pages(c, ws.movers, ws.holes, count);
}

int check_state(const ltv_page_state* s, bool lengths = true) {
  LTV_REQUIRE(s != nullptr, LTV_ERR_INVALID_ARG, "null state");
  LTV_REQUIRE(s->num_slots >= 0 && s->table_width >= 0 && s->num_pages >= 0 && s->page_size > 0 &&
                  s->table_stride >= s->table_width,
              LTV_ERR_INVALID_ARG, "bad state (slots=%d width=%d pages=%d page size=%d)",
              s->num_slots, s->table_width, s->num_pages, s->page_size);
  LTV_REQUIRE((int64_t)s->table_width * s->page_size < (int64_t(1) << 31), LTV_ERR_UNSUPPORTED,
              "a sequence's tokens must fit 31 bits");
  LTV_REQUIRE((s->num_slots == 0 || s->seq_lens || !lengths) &&
                  (s->num_pages == 0 || s->ref_counts) &&
                  (s->num_slots == 0 || s->table_width == 0 || s->page_table),
              LTV_ERR_INVALID_ARG, "null page table, lengths or reference counts");
  return LTV_OK;
}

int check_blocks(const ltv_page_blocks* b) {
  LTV_REQUIRE(b != nullptr, LTV_ERR_INVALID_ARG, "null blocks");
  LTV_REQUIRE(b->layers >= 0 && b->num_pages >= 0 && b->block_bytes >= 0, LTV_ERR_INVALID_ARG,
              "bad blocks (layers=%d pages=%d)", b->layers, b->num_pages);
  if (b->layers == 0 || b->num_pages == 0 || b->block_bytes == 0) return LTV_OK;
  LTV_REQUIRE(b->k && b->v, LTV_ERR_INVALID_ARG, "null pages");
  LTV_REQUIRE(aligned16(b->k) && aligned16(b->v) && b->block_bytes % 16 == 0 &&
                  b->k_page_bytes % 16 == 0 && b->v_page_bytes % 16 == 0 &&
                  b->k_layer_bytes % 16 == 0 && b->v_layer_bytes % 16 == 0,
              LTV_ERR_UNSUPPORTED, "pages must be 16-byte aligned blocks of a multiple of 16 bytes");
  return LTV_OK;
}

#define LTV_TRY(expr)              \
  do {                             \
    const int rc_ = (expr);        \
    if (rc_ != LTV_OK) return rc_; \
  } while (0)

// Pieces of `count` page copies, and workgroups for them.
int64_t copy_pieces(const ltv_page_blocks& b, int count) {
  const int64_t piece = (int64_t)kCopyPiece * 16;
  return (int64_t)count * b.layers * 2 * ((b.block_bytes + piece - 1) / piece);
}
int copy_grid(const ltv_page_blocks& b, int count) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(copy_pieces(b, count), kCopyGrid));
}
int check_copies(const ltv_page_blocks& b, int count) {
  LTV_REQUIRE(b.block_bytes < (int64_t(1) << 31) && copy_pieces(b, count) < (int64_t(1) << 31),
              LTV_ERR_UNSUPPORTED, "too many or too large pages to copy in a call");
  return LTV_OK;
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" int ltv_serving_abi_version(void) { return 1; }

extern "C" int ltv_paged_cache_append(int dtype, const void* k, const int64_t k_strides[3],
                                      const void* v, const int64_t v_strides[3], void* k_pages,
                                      const int64_t k_page_strides[3], void* v_pages,
                                      const int64_t v_page_strides[3],
                                      const ltv_paged_batch* batch, int NKVH, int D,
                                      void* stream) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  LTV_TRY(check_batch(batch));
  LTV_REQUIRE(NKVH >= 0 && D >= 0, LTV_ERR_INVALID_ARG, "bad shape (NKVH=%d D=%d)", NKVH, D);
  if (batch->B == 0 || batch->total == 0 || NKVH == 0 || D == 0 || batch->num_pages == 0 ||
      batch->num_slots == 0 || batch->table_width == 0)
    return LTV_OK;
  LTV_REQUIRE(k && v && k_pages && v_pages && k_strides && v_strides && k_page_strides &&
                  v_page_strides,
              LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(batch->B <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 sequences in a call");
  const int es = elem_size(dtype);
  AppendArgs a{PagedBatch(*batch), {(const char*)k, (const char*)v},
               {(char*)k_pages, (char*)v_pages}, {}, {}, NKVH, 0};
  uint64_t align = (uint64_t)k | (uint64_t)v | (uint64_t)k_pages | (uint64_t)v_pages |
                   (uint64_t)((int64_t)D * es);
  const int64_t* in_s[2] = {k_strides, v_strides};
  const int64_t* out_s[2] = {k_page_strides, v_page_strides};
  for (int w = 0; w < 2; ++w)
    for (int i = 0; i < 3; ++i) {
      a.ss[w][i] = in_s[w][i] * es;
      a.ps[w][i] = out_s[w][i] * es;
      align |= (uint64_t)a.ss[w][i] | (uint64_t)a.ps[w][i];
    }
  const bool wide = align % 16 == 0;
  a.units = wide ? D * es / 16 : D;
  LTV_REQUIRE(batch->total * NKVH * a.units < (int64_t(1) << 31), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  // (T is a hint with starts: the blocks stride over whatever there is)
  const int64_t units = (int64_t)std::max(batch->T, 1) * NKVH * a.units;
  const int blocks = (int)std::min<int64_t>((units + 255) / 256, 1024);
  const dim3 grid(blocks, batch->B, 2);
  const hipStream_t st = (hipStream_t)stream;
  if (wide)
    hipLaunchKernelGGL(append_kernel<uint4>, grid, dim3(256), 0, st, a);
  else if (es == 4)
    hipLaunchKernelGGL(append_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(append_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" size_t ltv_paged_cache_reserve_workspace_size(int n, int num_pages) {
  if (n <= 0 || num_pages < 0) return 0;
  return reserve_ws_ints(n, num_pages) * sizeof(int32_t);
}

extern "C" int ltv_paged_cache_reserve(const ltv_page_state* state, const ltv_page_blocks* blocks,
                                       const int32_t* slots, const int32_t* counts, int n,
                                       int32_t* status, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  LTV_TRY(check_state(state));
  LTV_TRY(check_blocks(blocks));
  LTV_REQUIRE(n > 0, LTV_ERR_INVALID_ARG, "no entries (n=%d)", n);
  LTV_REQUIRE(slots && counts && status && workspace, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(blocks->num_pages == state->num_pages, LTV_ERR_INVALID_ARG,
              "%d pages, %d reference counts", blocks->num_pages, state->num_pages);
  LTV_REQUIRE(workspace_bytes >= ltv_paged_cache_reserve_workspace_size(n, state->num_pages),
              LTV_ERR_WORKSPACE, "workspace too small");
  LTV_TRY(check_copies(*blocks, n));
  const State s = state_of(*state);
  ReserveWs ws;
  int32_t* w = reinterpret_cast<int32_t*>(workspace);
  ws.first = w;
  ws.plan = ws.first + n;
  ws.src = ws.plan + n;
  ws.dst = ws.src + n;
  ws.writers = ws.dst + n;
  ws.last = ws.writers + s.P;
  ws.count = ws.last + s.P;
  const hipStream_t st = (hipStream_t)stream;
  const bool wide = (int64_t)n * ((int64_t)s.W + 1) >= (int64_t(1) << 31);
  hipLaunchKernelGGL(wide ? reserve_kernel<long long> : reserve_kernel<int>, dim3(1),
                     dim3(kScanThreads), 0, st, s, slots, counts, n, ws, status);
  LTV_LAUNCH_CHECK();
  if (blocks->layers > 0 && blocks->block_bytes > 0 && state->num_pages > 0) {
    hipLaunchKernelGGL(copy_kernel, dim3(copy_grid(*blocks, n)), dim3(kCopyThreads), 0, st,
                       copy_args(*blocks), ws.src, ws.dst, ws.count, n);
    LTV_LAUNCH_CHECK();
  }
  return LTV_OK;
}

extern "C" int ltv_paged_cache_fork(const ltv_page_state* state, const int32_t* src,
                                    const int32_t* dst, int n, void* stream) {
  LTV_TRY(check_state(state));
  LTV_REQUIRE(n >= 0, LTV_ERR_INVALID_ARG, "bad number of entries %d", n);
  if (n == 0 || state->num_slots == 0) return LTV_OK;
  LTV_REQUIRE(src && dst, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(n <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 entries");
  const int blocks = std::max(1, std::min((state->table_width + 255) / 256, 64));
  hipLaunchKernelGGL(fork_kernel, dim3(blocks, n), dim3(256), 0, (hipStream_t)stream,
                     state_of(*state), src, dst);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" int ltv_paged_cache_free(const ltv_page_state* state, const int32_t* slots, int n,
                                    void* stream) {
  LTV_TRY(check_state(state));
  LTV_REQUIRE(n >= 0, LTV_ERR_INVALID_ARG, "bad number of entries %d", n);
  if (n == 0 || state->num_slots == 0) return LTV_OK;
  LTV_REQUIRE(slots, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(n <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 entries");
  const int blocks = std::max(1, std::min((state->table_width + 255) / 256, 64));
  hipLaunchKernelGGL(free_kernel, dim3(blocks, n), dim3(256), 0, (hipStream_t)stream,
                     state_of(*state), slots);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" size_t ltv_paged_cache_reorder_workspace_size(int n, int table_width) {
  if (n <= 0 || table_width < 0) return 0;
  return (size_t)n * ((size_t)table_width + 1) * sizeof(int32_t);
}

extern "C" int ltv_paged_cache_reorder(const ltv_page_state* state, const int32_t* slots,
                                       const int32_t* src, int n, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  LTV_TRY(check_state(state));
  LTV_REQUIRE(n >= 0, LTV_ERR_INVALID_ARG, "bad number of entries %d", n);
  if (n == 0 || state->num_slots == 0) return LTV_OK;
  LTV_REQUIRE(slots && src, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(n <= 65535, LTV_ERR_UNSUPPORTED, "more than 65,535 entries");
  LTV_REQUIRE(workspace && aligned16(workspace) &&
                  workspace_bytes >= ltv_paged_cache_reorder_workspace_size(n, state->table_width),
              LTV_ERR_WORKSPACE, "workspace too small");
  const hipStream_t st = (hipStream_t)stream;
  if (n <= kReorderInts >> 2) {
    // (two entries of a thread, so that many workgroups share a call; 384 rows of 502 pages 9.4 us
    // with 16 columns to each)
    int log_cols = 6;
    while (log_cols > 2 && n << log_cols > 2 * kReorderThreads) --log_cols;
    const int groups = (int)(((int64_t)state->table_width + (1 << log_cols) - 1) >> log_cols);
    hipLaunchKernelGGL(reorder_kernel, dim3(std::max(1, groups)), dim3(kReorderThreads), 0, st,
                       state_of(*state), slots, src, n, log_cols);
    LTV_LAUNCH_CHECK();
    return LTV_OK;
  }
  int32_t* lens = reinterpret_cast<int32_t*>(workspace);
  int32_t* rows = lens + n;
  const dim3 grid(std::max(1, std::min((state->table_width + 255) / 256, 64)), n);
  hipLaunchKernelGGL(reorder_read_kernel, grid, dim3(256), 0, st, state_of(*state), slots, src,
                     rows, lens);
  LTV_LAUNCH_CHECK();
  hipLaunchKernelGGL(reorder_write_kernel, grid, dim3(256), 0, st, state_of(*state), slots, src,
                     (const int32_t*)rows, (const int32_t*)lens);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" int ltv_paged_cache_copy(const ltv_page_blocks* blocks, const int32_t* src,
                                    const int32_t* dst, int n, void* stream) {
  LTV_TRY(check_blocks(blocks));
  LTV_REQUIRE(n >= 0, LTV_ERR_INVALID_ARG, "bad number of entries %d", n);
  if (n == 0 || blocks->layers == 0 || blocks->block_bytes == 0 || blocks->num_pages == 0)
    return LTV_OK;
  LTV_REQUIRE(src && dst, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_TRY(check_copies(*blocks, n));
  hipLaunchKernelGGL(copy_kernel, dim3(copy_grid(*blocks, n)), dim3(kCopyThreads), 0,
                     (hipStream_t)stream, copy_args(*blocks), src, dst, (const int32_t*)nullptr,
                     n);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

extern "C" size_t ltv_paged_cache_compact_workspace_size(int num_pages) {
  if (num_pages < 0) return 0;
  return compact_ws_ints(num_pages) * sizeof(int32_t);
}

extern "C" int ltv_paged_cache_compact(const ltv_page_state* state, const ltv_page_blocks* blocks,
                                       int32_t* live, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  LTV_TRY(check_state(state, false));
  LTV_TRY(check_blocks(blocks));
  LTV_REQUIRE(live && workspace, LTV_ERR_INVALID_ARG, "null pointer");
  LTV_REQUIRE(blocks->num_pages == state->num_pages, LTV_ERR_INVALID_ARG,
              "%d pages, %d reference counts", blocks->num_pages, state->num_pages);
  LTV_REQUIRE(workspace_bytes >= ltv_paged_cache_compact_workspace_size(state->num_pages),
              LTV_ERR_WORKSPACE, "workspace too small");
  LTV_TRY(check_copies(*blocks, std::max(1, state->num_pages / 2)));
  const State s = state_of(*state);
  CompactWs ws;
  ws.place = reinterpret_cast<int32_t*>(workspace);
  ws.movers = ws.place + s.P;
  ws.holes = ws.movers + s.P;
  ws.count = ws.holes + s.P;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kScanThreads), 0, st, s, ws, live);
  LTV_LAUNCH_CHECK();
  hipLaunchKernelGGL(compact_move_kernel, dim3(copy_grid(*blocks, std::max(1, s.P / 2))),
                     dim3(kCopyThreads), 0, st, copy_args(*blocks), s, ws);
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
