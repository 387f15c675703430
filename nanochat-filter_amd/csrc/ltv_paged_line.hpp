// What the kernels of attention over a paged cache share, whatever the pages hold: a call's row
// tiles laid on a line and cut into equal ranges, the rows that are computed one by one, and
// the joining of the tiles that were cut.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ltv_paged.hpp"

namespace ltv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  PagedBatch batch;
  const char* q;
  const char* k;
  const char* v;
  char* out;
  float* lse;
  float* part;                // partial o, then (m, l), of the tiles that are cut
  int64_t qs[3], os[3];       // bytes
  int64_t kh, vh;             // bytes from head to head of the pages
  uint32_t kp, ks, vp, vs;    // 16-byte units from page to page and row to row
  int NH, NKVH, D, g;
  int q_aligned;
  int all_rests;              // of probabilities
  int scalar_pages;           // load_full: pages are multiples of 16 rows
  float scale;                // with log2(e)
  int log_group, ranges;      // log2 of the workgroups side by side, and how many such groups
  int least;                  // shortest range
  int unit;                   // log2 of the blocks of keys in a unit of length
  int group_tokens, slope;    // tokens of a group's row tiles; units that each is longer by
  int extra;                  // units that a group's begin counts for
  int log_rows;               // of a row tile
  int part_tile;              // rows of a partial tile, 0: none is cut
  PageDiv by_g, by_ranges;    // divisions by g and by the number of ranges
  int64_t part_rows;
  int* head;                  // how many ranges the call came to
  struct Cut* cuts;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Nothing is moved across: the tile's loop is written in the order that it is to run in,
// reads from LDS well ahead of the products that take them and exponentials between the
// products.  (Left to itself the compiler puts each read right before its product.)
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ uint32_t lds_address(uint4* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *(__attribute__((address_space(3))) const V*)(uintptr_t)at;
}

__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ float across_halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The sum of x over the lanes up to each: within rows of 16 by shifts, then the rows' last.
__device__ __forceinline__ uint32_t wave_sum_up_to(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// An entry of a page table, through the scalar cache (col and table are the same for all lanes).
__device__ __forceinline__ int page_at(const int32_t* table, int col) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(table + col);
}

// (row numbers stay below 2^30: divisions of 64 bits would take longer than small calls)
__device__ __forceinline__ int over(int a, int b) { return (int)((unsigned)a / (unsigned)b); }

// The line.  A sequence's row tiles are taken in groups of 2^a.log_group that workgroups of
// one XCD work on side by side, so that its L2 holds what they read for all but the first:
// tiles of one k/v head, which read the same keys, or where it has fewer, of several heads.
// A group is as long as the blocks of keys (of one tile in LDS) of its longest row tile, in
// units of 2^a.unit blocks, about: c0, and slope more for each group of the head.
struct Line {
  int tiles, heads;  // row tiles, heads of a group
  int groups;        // of a head
  int rounds;        // times that many heads, all together
  uint32_t c0, head, all;

  __device__ __forceinline__ uint32_t before(const AttnArgs& a, int j) const {
    const uint32_t k = j;  // (the product's half modulo 2^32, whatever k is)
    return k * c0 + a.slope * (k % 2 ? (k - 1) / 2 * k : k / 2 * (k - 1));
  }
  template <int KT>
  static __device__ __forceinline__ Line of(const AttnArgs& a, int n, int len) {
    Line u{0, 1, 0, 0, 0, 0, 0};
    if (n <= 0) return u;
    u.tiles = (n * a.g + (1 << a.log_rows) - 1) >> a.log_rows;
    const int several = u.tiles == 1 ? a.log_group : u.tiles == 2 && a.log_group == 2 ? 1 : 0;
    u.heads = 1 << several;
    u.groups = (u.tiles + (1 << a.log_group) - 1) >> a.log_group;
    u.rounds = (a.NKVH + u.heads - 1) >> several;
    const int past = max(len - n, 0);
    u.c0 = max(1, (min(len, past + min(n, a.group_tokens)) + KT - 1) / KT >> a.unit) + a.extra;
    u.head = u.before(a, u.groups);
    u.all = u.rounds * u.head;
    return u;
  }
};

// Keys that the last row of a row tile sees, and the block of keys at which a cut at f of
// the tile's c units is, the first `extra` of which stand for no keys.
__device__ __forceinline__ int keys_of(const AttnArgs& a, const PagedSeq& s, int tile) {
  const int last = a.by_g.quot(min((tile + 1) << a.log_rows, s.n * a.g) - 1);
  return a.batch.P > 0 && a.batch.W > 0 ? max(s.len - s.n + last + 1, 0) : 0;
}
__device__ __forceinline__ int cut_at(uint32_t f, uint32_t c, int blocks, uint32_t extra) {
  if (f >= c) return blocks;
  if (f <= extra) return 0;
  return min(blocks, (int)fmaf((float)(f - extra),
                               (float)blocks * __builtin_amdgcn_rcpf((float)(c - extra)), 0.5f));
}

// Where the ranges begin: `length` apart, every other one by `lead` later.
struct Ranges {
  uint32_t length, lead;
  int count;
  __device__ __forceinline__ uint32_t begin(int i) const {
    return i * length + (i & 1 ? lead : 0);
  }
  __device__ __forceinline__ int of(uint32_t x) const {  // .. which x is in
    const int i = over(x, length);
    return min(i - ((i & 1) && x < begin(i)), count - 1);
  }
};

// A row tile whose first cut is a workgroup's begin, for the joining kernel.
struct Cut {
  int rows;           // 0: none
  int b, kvh, token;  // token: of the sequence's first, in packed rows
  int tile, last;     // last: range with a piece of it
  int pad[2];
};

// Rows of partials (D values each; behind them all, each row's m and l): two row tiles for
// each workgroup, of the piece that continues a tile and of the one that begins the last.
__device__ __forceinline__ int64_t part_at(const AttnArgs& a, int range, int member, bool begins) {
  return ((int64_t)((range << a.log_group) + member) * 2 + begins) * a.part_tile;
}
__device__ __forceinline__ float2* part_ml(const AttnArgs& a) {
  return reinterpret_cast<float2*>(a.part + a.part_rows * a.D);
}

// Rows row0 .. row_end - 1 of a workgroup over keys begin .. end - 1, each key that a row
// does not see left alone altogether: the way of tiles with infinite or NaN values among
// those that some rows do not see.  Groups of sixteen lanes take a row's keys in turn, a lane
// holding eight channels, which Pages reads (chunk c of a key in its page).  part0: the partials
// of row0, or -1.  shift: values come as 2^-shift of what they are, so that their sum stays in
// range; (m, l, o) are left as the same (m + shift, l 2^-shift, o 2^-shift).
template <typename T, int THREADS, typename Pages>
__device__ __forceinline__ void rows_one_by_one(const AttnArgs& a, const PagedSeq& s, int b,
                                                int kvh, int row0, int row_end, int begin, int end,
                                                int64_t part0, float* lds, int shift = 0) {
#pragma clang fp contract(off)  // (x - base below must not be a fused form of the product)
  float* lds_m = lds;
  constexpr int G = THREADS / 16;
  float* lds_l = lds + G;
  float* lds_o = lds + 2 * G;  // G x 128
  const int c = threadIdx.x & 15, gi = threadIdx.x >> 4;
  const bool on = c * 8 < a.D;
  for (int row = row0; row < row_end; ++row) {
    const int t = a.by_g.quot(row), h = kvh * a.g + row - t * a.g;
    const int last = min(end - 1, s.len - s.n + t);
    const int64_t trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;
    const char* q = a.q + (a.batch.starts != nullptr ? trow * a.qs[1]
                                                     : b * a.qs[0] + t * a.qs[1]) + h * a.qs[2];
    float qf[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[e] = on ? io_traits<T>::load(reinterpret_cast<const T*>(q) + c * 8 + e) : 0.0f;
      o[e] = 0.0f;
    }
    for (int j = begin + gi; j <= last; j += G) {
      const int col = a.batch.div.quot(j), page = s.table[col];
      if (page < 0 || page >= a.batch.P) continue;
      const uint32_t in = (uint32_t)(j - col * a.batch.div.size);
      float x = 0.0f;
      float kv[8];
      if (on) {
        Pages::keys(a, kvh, page, in, c, kv);
        for (int e = 0; e < 8; ++e) x = fmaf(qf[e], kv[e], x);
      }
      for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
      x *= a.scale;
      const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.0f : mn;
      const float was = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(x - base);
      l = fmaf(l, was, p);
      m = mn;
      if (on) {
        Pages::values(a, kvh, page, in, c, kv, shift);
        for (int e = 0; e < 8; ++e) o[e] = fmaf(p, kv[e], o[e] * was);
      }
    }
    __syncthreads();
    if (c == 0) {
      lds_m[gi] = m;
      lds_l[gi] = l;
    }
    for (int e = 0; e < 8; ++e) lds_o[gi * 128 + c * 8 + e] = o[e];
    __syncthreads();
    float mx = -INFINITY;
    for (int i = 0; i < G; ++i) mx = fmaxf(mx, lds_m[i]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, acc[128 / THREADS + 1] = {};
    const int d0 = threadIdx.x;
    for (int i = 0; i < G; ++i) {
      // (a group without keys has weight 0)
      const float w = lds_m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lds_m[i] - base);
      sum = fmaf(lds_l[i], w, sum);
#pragma unroll
      for (int e = 0, d = d0; d < 128; ++e, d += THREADS) acc[e] = fmaf(lds_o[i * 128 + d], w, acc[e]);
    }
    if (part0 >= 0) {
      const int64_t at = part0 + row - row0;
#pragma unroll
      for (int e = 0, d = d0; d < 128; ++e, d += THREADS)
        if (d < a.D) a.part[at * a.D + d] = acc[e];
      if (d0 == 0) part_ml(a)[at] = make_float2(mx + shift, ldexpf(sum, -shift));
    } else {
      char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                     : b * a.os[0] + t * a.os[1]) + h * a.os[2];
#pragma unroll
      for (int e = 0, d = d0; d < 128; ++e, d += THREADS)
        if (d < a.D)
          io_traits<T>::store(reinterpret_cast<T*>(out) + d,
                              sum == 0.0f ? 0.0f : ldexpf(acc[e] / sum, shift));
      if (d0 == 0 && a.lse != nullptr)
        a.lse[trow * a.NH + h] = sum == 0.0f ? -INFINITY
                                             : (mx + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

// A workgroup's range of the line: piece(s, b, kvh, tile, begin, end, part0) computes keys begin ..
// end of a row tile, into its rows of the output or the partials from part0 on (-1: none).  KT:
// keys of a block, ROWS: of a row tile, GRID: workgroups that the card holds; FEW: one wavefront,
// and many sequences to a thread.  Args: AttnArgs, or a reference, as leaves the kernel's loop over
// tiles with fewer numbers put aside for scalar registers (a long prompt over 16-bit pages 1,254 us
// with a reference and 1,155 with a copy; over 4-bit pages they are alike).
template <int KT, bool FEW, int THREADS, int ROWS, int GRID, typename Args, typename Piece>
__device__ __forceinline__ void walk_line(Args a, Piece piece) {
  constexpr int WAVES = THREADS / 64;
  // The lengths of all sequences, a run of them to each thread, and their sum.
  __shared__ uint32_t sums[WAVES];
  __shared__ struct { PagedSeq s; int b; uint32_t at; } found;  // the sequence of a range's begin
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (a.batch.B + THREADS - 1) / THREADS;
  const int b0 = min((int)threadIdx.x * per, a.batch.B), b1 = min(b0 + per, a.batch.B);
  uint32_t mine = 0;
  PagedSeq q{a.batch.table, 0, 0, 0};
  for (int i = b0; i < b1; ++i) {
    q = paged_seq(a.batch, i);
    mine += Line::of<KT>(a, q.n, q.len).all;
  }
  uint32_t upto = wave_sum_up_to(mine);
  if ((threadIdx.x & 63) == 63) sums[wave] = upto;
  if (threadIdx.x == 0) {
    found.s = q;
    found.b = 0;
    found.at = 0;
  }
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) upto += sums[w];
    all += sums[w];
  }
  all = __builtin_amdgcn_readfirstlane(all);
  Ranges line;
  line.length = max(a.least, a.by_ranges.quot(all + a.ranges - 1));
  line.count = min(over(all + line.length - 1, line.length), a.ranges);
  // Of the two workgroups of a compute unit the older is served first where the products
  // bound them, and had ended with a fifth of the other's work left: it gets more of it
  // (a long prompt 1,225 us with equal ranges, 1,187 with these).
  const bool full = a.log_group > 0 && line.count << a.log_group == GRID;
  line.lead = full ? line.length / 8 : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.head = line.count;
  // Workgroup w runs on XCD w % 8: consecutive ranges stay on one.
  const int per_xcd = (line.count + 7) / 8, local = blockIdx.x >> 3 >> a.log_group;
  const int range = (blockIdx.x & 7) * per_xcd +
                    (!full ? local : local < per_xcd / 2 ? local * 2 : local * 2 - per_xcd + 1);
  const int member = (blockIdx.x >> 3) & ((1 << a.log_group) - 1);
  if (local >= per_xcd || range >= line.count) return;
  if (threadIdx.x == 0) a.cuts[(range << a.log_group) + member].rows = 0;  // (until it has one)
  const uint32_t x0 = line.begin(range), x1 = min(line.begin(range + 1), all);
  if (x0 >= all) return;
  if (x0 >= upto - mine && x0 < upto) {
    uint32_t at = upto - mine;
    int i = b0;
    if (!FEW && per > 1)
      for (;; ++i) {
        q = paged_seq(a.batch, i);
        const uint32_t here = Line::of<KT>(a, q.n, q.len).all;
        if (x0 - at < here || i == b1 - 1) break;
        at += here;
      }
    found.s = q;
    found.b = i;
    found.at = at;
  }
  __syncthreads();
  auto uniform = [](auto x) {  // (from LDS, into scalar registers)
    static_assert(sizeof(x) % 4 == 0, "whole words");
    int w[sizeof(x) / 4];
    __builtin_memcpy(w, &x, sizeof(x));
#pragma unroll
    for (int i = 0; i < (int)sizeof(x) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
    __builtin_memcpy(&x, w, sizeof(x));
    return x;
  };
  int b = uniform(found.b);
  uint32_t at = uniform(found.at);  // of the group on the line
  if (FEW && per > 1) {
    // Which of the thread's sequences, one to a lane.  (2,048 of them 184 us searched by the
    // thread, 176 so; in the other shape, with a fourth of them to a thread, it only adds
    // instructions to every start: chunks among decoding sequences 103 and 104.)
    const int end = min(b + per, a.batch.B), lane = threadIdx.x;
    __syncthreads();  // (found is read)
    for (;; b += 64) {
      PagedSeq mine{a.batch.table, 0, 0, 0};
      if (b + lane < end) mine = paged_seq(a.batch, b + lane);
      const uint32_t here = Line::of<KT>(a, mine.n, mine.len).all, to = wave_sum_up_to(here);
      const uint64_t past = __ballot(x0 - at < to);
      if (past == 0 && b + 64 < end) {
        at += __builtin_amdgcn_readlane(to, 63);
        continue;
      }
      const int l = past == 0 ? 0 : __builtin_ctzll(past);
      if (lane == l) {
        found.s = mine;
        found.b = b + l;
        found.at = at + to - here;
      }
      break;
    }
    __syncthreads();
    b = uniform(found.b);
    at = uniform(found.at);
  }
  PagedSeq s{uniform(found.s.table), uniform(found.s.len), uniform(found.s.n),
             uniform(found.s.row0)};
  Line u = Line::of<KT>(a, s.n, s.len);
  if (u.all == 0) return;  // (starts that do not ascend)
  int round = over(x0 - at, u.head), group = 0;
  at += round * u.head;
  for (int hi = u.groups - 1; group < hi;) {
    const int mid = (group + hi + 1) >> 1;
    if (u.before(a, mid) <= x0 - at) group = mid; else hi = mid - 1;
  }
  at += u.before(a, group);
  for (uint32_t x = x0;;) {
    // units from .. to of a group's c
    const uint32_t c = u.c0 + a.slope * group;
    const uint32_t from = x - at, to = min(x1 - at, c);
    // (several heads: one or two tiles of each)
    const int k = u.heads == 1 ? 0 : member >> (u.tiles - 1);
    const int kvh = round * u.heads + k;
    const int tile = u.heads == 1 ? (group << a.log_group) + member : member & (u.tiles - 1);
    const bool on = k < u.heads && (unsigned)kvh < (unsigned)a.NKVH && tile < u.tiles;
    // (a sequence of more rows than there is room for is not cut)
    const int rows = s.n * a.g;
    const bool cuts = min(rows, ROWS) <= a.part_tile;
    if (on && (cuts || from == 0)) {
      const bool whole = !cuts || (from == 0 && to == c);
      const int keys = keys_of(a, s, tile), blocks = (keys + KT - 1) / KT;
      const int begin = whole ? 0 : cut_at(from, c, blocks, a.extra) * KT;
      const int end = whole || to == c ? keys : min(keys, cut_at(to, c, blocks, a.extra) * KT);
      if (x == x0 && from > 0 && at >= line.begin(range - 1) && threadIdx.x == 0)
        a.cuts[(range << a.log_group) + member] =
            Cut{min(rows - tile * ROWS, ROWS), b, kvh, (int)s.row0, tile,
                line.of(at + c - 1), {}};
      if (!whole && begin >= end) {  // (a piece of no keys)
        const int64_t part0 = part_at(a, range, member, from == 0);
        if ((int)threadIdx.x < min(rows - tile * ROWS, ROWS))
          part_ml(a)[part0 + threadIdx.x] = make_float2(-INFINITY, 0.0f);
      } else {
        piece(s, b, kvh, tile, begin, end, whole ? -1 : part_at(a, range, member, from == 0));
      }
    }
    x = at + to;
    if (x >= x1) return;
    at += c;
    ++group;
    // (taken anew, so that it is not kept in registers through a piece)
    s = paged_seq(a.batch, b);
    u = Line::of<KT>(a, s.n, s.len);
    if (group == u.groups) {
      group = 0;
      ++round;
    }
    while (round >= u.rounds) {
      if (++b >= a.batch.B) return;
      s = paged_seq(a.batch, b);
      u = Line::of<KT>(a, s.n, s.len);
      round = 0;
    }
  }
}

// Joins the pieces of the row tiles that were cut, 32 lanes to a row and four channels to a
// lane.  Of few pieces 32 lanes take all of a row, of many the eight groups of a workgroup
// share a row's.  It is all latency: the record of the cut, then the partials of four pieces
// at a time.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a, int rows_each) {
  constexpr int G = 8;  // groups
  __shared__ float lds_o[G][128];
  __shared__ float2 lds_ml[G];
  const int range = blockIdx.x >> a.log_group, member = blockIdx.x & ((1 << a.log_group) - 1);
  const Cut cut = a.cuts[blockIdx.x];
  if (range >= *a.head) return;
  const int first = range - 1, pieces = cut.last - first + 1;
  const int row0 = blockIdx.y * rows_each, row_end = min(cut.rows, row0 + rows_each);
  if (row0 >= row_end) return;
  const bool share = pieces > (rows_each == 1 ? 4 : 16);
  const int lane = threadIdx.x & 31, gi = threadIdx.x >> 5;
  const bool on = lane * 4 < a.D;
  for (int row = row0 + (share ? 0 : gi); row < row_end; row += share ? 1 : G) {
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = first + (share ? gi : 0); p0 <= cut.last; p0 += 4 * (share ? G : 1)) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + i * (share ? G : 1), pp = min(p, cut.last);
        const int64_t at = part_at(a, pp, member, pp == first) + row;
        ml[i] = part_ml(a)[at];
        v[i] = on ? *reinterpret_cast<const float4*>(a.part + at * a.D + lane * 4)
                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // (a piece without keys has no sums; a NaN is one)
        if (p > cut.last || ml[i].y == 0.0f) {
          ml[i] = make_float2(-INFINITY, 0.0f);
          v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 4; ++i) mn = fmaxf(mn, ml[i].x);
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float was = __builtin_amdgcn_exp2f(m - base);
      m = mn;
      l *= was;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= was;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = __builtin_amdgcn_exp2f(ml[i].x - base);
        l = fmaf(ml[i].y, w, l);
        o[0] = fmaf(v[i].x, w, o[0]);
        o[1] = fmaf(v[i].y, w, o[1]);
        o[2] = fmaf(v[i].z, w, o[2]);
        o[3] = fmaf(v[i].w, w, o[3]);
      }
    }
    if (share) {
      __syncthreads();  // (the row before is read)
#pragma unroll
      for (int e = 0; e < 4; ++e) lds_o[gi][lane * 4 + e] = o[e];
      if (lane == 0) lds_ml[gi] = make_float2(m, l);
      __syncthreads();
      if (gi != 0) continue;
#pragma unroll
      for (int i = 0; i < G; ++i) m = fmaxf(m, lds_ml[i].x);
      const float base = m == -INFINITY ? 0.0f : m;
      l = o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float w = __builtin_amdgcn_exp2f(lds_ml[i].x - base);
        l = fmaf(lds_ml[i].y, w, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(lds_o[i][lane * 4 + e], w, o[e]);
      }
    }
    const int r = (cut.tile << a.log_rows) + row, t = a.by_g.quot(r), h = cut.kvh * a.g + r - t * a.g;
    const int64_t trow = (a.batch.starts != nullptr ? cut.token : (int64_t)cut.b * a.batch.T) + t;
    char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                   : cut.b * a.os[0] + t * a.os[1]) + h * a.os[2];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (on) {
      if constexpr (sizeof(T) == 2)
        reinterpret_cast<uint2*>(out)[lane] =
            make_uint2(cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv));
      else
        reinterpret_cast<float4*>(out)[lane] =
            make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
    if (lane == 0 && a.lse != nullptr)
      a.lse[trow * a.NH + h] =
          l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// How a call is cut.
struct AttnPlan {
  bool few;
  int log_rows, group, ranges, least, unit, group_tokens, slope, extra, part_tile;
  bool joins, all_rests;
  int64_t part_rows;
  size_t bytes, cuts_at;
};

// What a kernel is made for, and what was found best for it.
struct LineShape {
  int keys, log_rows;  // of a block, of a row tile
  int grid;            // workgroups that the card holds
  int group;           // row tiles side by side
  int least;           // blocks of the shortest range
  bool few;
};

AttnPlan plan_line(const ltv_paged_batch& b, int NH, int NKVH, int D, int max_len,
                   const LineShape& shape) {
  AttnPlan p{};
  p.few = shape.few;
  p.log_rows = shape.log_rows;
  p.group = shape.group;
  p.least = shape.least;
  const int KT = shape.keys;
  const int64_t tile = int64_t(1) << shape.log_rows, group_rows = p.group * tile;
  const int64_t g = NH / NKVH, rows = std::max(b.T, 1) * g, tiles = (rows + tile - 1) / tile;
  p.group_tokens = (int)((group_rows + g - 1) / g);
  // (where no sequence can have more than a block of keys none is cut)
  const int64_t keys = (int64_t)b.table_width * b.page_size;
  p.joins = keys > KT;
  p.part_tile = p.joins ? (int)std::min<int64_t>(rows, tile) : 0;
  // (fewer, if the call has no more tiles than that)
  const int64_t groups =
      NKVH * std::min((tiles + p.group - 1) / p.group * b.B, b.total * g / group_rows + b.B);
  const int64_t most = groups * ((std::max(max_len, 1) + KT - 1) / KT);
  p.ranges = (int)std::min<int64_t>(shape.grid / p.group, (most + p.least - 1) / p.least);
  p.ranges = std::max(8, (p.ranges + 7) / 8 * 8);
  // Positions on the line have 32 bits: units of more blocks where it could be longer than
  // 2^30, whatever the lengths are.
  const double bound = (double)NKVH * ((double)b.total * g / group_rows + b.B) *
                       ((double)(keys + b.total) / KT + 64);
  p.unit = 0;
  while (bound / (double)(int64_t(1) << p.unit) > (double)(1 << 30)) ++p.unit;
  p.slope = (int)(group_rows / g / KT) >> p.unit;
  // What a piece costs beside its keys -- its rows, the first tile's way, the remainders that
  // the first tiles take, its partials -- counted in blocks: four, or none where few rows have
  // a range for every few blocks.  (Without and with it: chunks mixed with decoding 110 and 98
  // us, float32 chunks 50 and 48, a ragged decode step 282 and 261; a small one 17.6 and, with
  // one block, 18.4.  Two, four and eight for 256 sequences of up to 2,000 tokens 222, 219, 224.)
  p.extra = (p.few || rows > 32 || most > 8 * shape.grid ? 4 : 0) >> p.unit;
  const int64_t n = (int64_t)p.ranges * p.group;
  p.part_rows = n * 2 * p.part_tile;
  p.cuts_at = (size_t)p.part_rows * (D + 2) * sizeof(float);
  p.bytes = p.cuts_at + n * sizeof(Cut) + 16;
  return p;
}

}  // namespace
}  // namespace ltv
