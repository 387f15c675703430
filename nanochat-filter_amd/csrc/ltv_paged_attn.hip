// Attention of new tokens over a paged cache.
//
//   out[row] = sum_j p_j v_j,  p = softmax_{j <= pos(row)}(scale q[row] . k_j)
//
// One pass over the keys with the running maximum m and sum l of each row's softmax:
// for a tile of keys, s = scale log2(e) K q, m' = max(m, max s), p = 2^(s - m'),
// l = l 2^(m - m') + sum p, o = o 2^(m - m') + V^T p, and out = o / l at the end.
//
// Rows.  A sequence's n tokens times the g = NH / NKVH query heads of one k/v head are
// its rows, token-major: they share every key, so a decode step of a group of heads
// reads its keys once.  A workgroup has 128 rows, 32 for each of four wavefronts (or one
// wavefront, where many sequences have few rows each).
//
// Layout of the products (32 x 32 MFMA blocks).  The scores are computed as S^T = K Q^T:
// a lane then holds 16 keys of one row, so maximum and sum are taken in the lane and
// once across the two half-wavefronts, and its values are, without any exchange, the
// right-hand operand of O^T = V^T P^T: the order of the keys within a product is free
// as long as V^T is read in the same one (ds_read_b64_tr_b16 transposes four keys of a
// column at a time).  Both tiles are shared by the wavefronts through LDS, two buffers
// deep: the next tile is on its way, straight into LDS, while this one is computed.
//
// Work.  All row tiles of a call, each as long as its keys, are laid on a line, and the
// line is cut into equal ranges, one for each workgroup that the card holds at a time: no
// workgroup is empty or ends late, whatever mixture of lengths a call has.  The line is made
// on the device, which knows the lengths.  A range begins and ends within a row tile as it
// comes; a second kernel joins the (m, l, o) of the tiles that were cut.  (Every sequence cut
// into the same number of chunks instead, in the same calls: 322 us and 260 now for a decode
// step with one very long context, 144 and 98 for chunks among decoding sequences, 1,500 and
// 1,195 for the last chunk of a long prompt.)
//
// What bounds it.  One new token of each sequence: memory, 64 sequences of 8,000 tokens at 5.7
// TB/s (a copy reaches 5.0, half of it writes).  Long chunks: the matrix unit, busy 46 % of the
// cycles, and the vector unit, issuing in 51 %, in turn: 12,289 tokens over 32,289 at 803 to 853
// TFLOP/s where a plain product of two 8,192 x 8,192 matrices reaches 1,121.  Little work: latency, 2 us until a workgroup has found its
// range, 4 until its first tile has landed, 2 to write, 3 to join.
#include <algorithm>
#include <type_traits>

#include "ltv_gemm_dma.hpp"
#include "ltv_paged.hpp"

namespace ltv {
namespace {

// A workgroup: four wavefronts and tiles of 64 keys (float32: 32), two to a compute unit; of
// few rows, which one wavefront holds, that one and tiles of 32 keys, four to a unit.
template <typename T, bool FEW>
struct AttnShape {
  static constexpr int kWaves = FEW ? 1 : 4, kThreads = kWaves * 64, kRows = kWaves * 32;
  static constexpr int kGrid = FEW ? 1024 : 512;  // workgroups that the card holds
  static constexpr int kKeys = FEW || sizeof(T) == 4 ? 32 : 64;  // of a tile
};
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

// What differs by element type.  A chunk is 16 bytes of a row.
template <typename T>
struct AttnType;

template <>
struct AttnType<bf16_t> {
  static constexpr int kChunk = 8;  // elements
  // S^T += K Q^T over 16 channels: a lane's k and q chunk hold channels 8 (lane / 32) ..
  static __device__ __forceinline__ f32x16 scores(u32x4_t k, uint4 q, f32x16 s) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                   __builtin_bit_cast(bf16x8_t, q), s, 0, 0, 0);
  }
};

template <>
struct AttnType<float> {
  static constexpr int kChunk = 4;
  static __device__ __forceinline__ f32x16 scores(u32x4_t k, uint4 q, f32x16 s) {
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.x), __uint_as_float(q.x), s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.y), __uint_as_float(q.y), s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.z), __uint_as_float(q.z), s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.w), __uint_as_float(q.w), s, 0, 0, 0);
    return s;
  }
};

// Shape of a tile in LDS: rows of DP channels (D padded with zeros), unpadded; chunk c of
// row r sits in a slot chosen so that the lanes of one read fall on different banks.
//   K: 16 consecutive rows, one chunk each (ds_read_b128).
//   V, bfloat16: four rows, 64 bytes each (ds_read_b64_tr_b16).
//   V, float32: two rows four apart, 128 bytes each (ds_read_b32).
template <typename T, int DP, bool FEW>
struct AttnTile {
  static constexpr int kKeys = AttnShape<T, FEW>::kKeys, kAttnThreads = AttnShape<T, FEW>::kThreads;
  static constexpr int kChunks = DP / AttnType<T>::kChunk;     // of a row
  static constexpr int kPhase = kChunks < 16 ? 16 / kChunks : 1;  // rows of 256 bytes
  static constexpr int kUnits = kKeys * kChunks;               // chunks of a tile
  static constexpr int kLoads = kUnits / kAttnThreads;         // of a thread
  static_assert(kUnits % kAttnThreads == 0, "a tile is loaded by all threads alike");
  static __device__ __forceinline__ int k_swizzle(int r) {
    return (r / kPhase) & 15 & (kChunks - 1);
  }
  static __device__ __forceinline__ int v_swizzle(int r) {
    if constexpr (sizeof(T) == 4) return ((r >> 2) & 1) * 8;
    return ((r / kPhase) & (4 / kPhase - 1)) * 4;
  }
};

__device__ const uint4 kZeros = {0, 0, 0, 0};

__device__ __forceinline__ uint32_t lds_address(uint4* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *(__attribute__((address_space(3))) const V*)(uintptr_t)at;
}

// One wavefront's 16 bytes per lane from `from` into LDS at `to` + 16 lane (`to` uniform).
// Inline assembly, as in the projection's kernels: the compiler would wait for a builtin's
// load before the next read of either buffer.  It has no output register; the wait is
// wait_vmcnt and a barrier.  The nop covers the write of M0.
__device__ __forceinline__ void load_lds16(uint4* to, const char* from) {
  const uint32_t base = lds_address(to);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(base) : "memory");
}

// The same from a uniform address and an offset of the lane.
__device__ __forceinline__ void load_lds16(uint4* to, const char* from, uint32_t offset) {
  const uint32_t base = lds_address(to);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(from),
               "{m0}"(base) : "memory");
}

__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Whether any of a chunk's elements is infinite or NaN (all exponent bits set).
__device__ __forceinline__ bool any_nonfinite(uint4 x, bf16_t) {
  bool bad = false;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}
__device__ __forceinline__ bool any_nonfinite(uint4 x, float) {
  bool bad = false;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
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
// holding eight channels.  part0: the partials of row0, or -1.
template <typename T, int THREADS>
__device__ __forceinline__ void rows_one_by_one(const AttnArgs& a, const PagedSeq& s, int b,
                                                int kvh, int row0, int row_end, int begin, int end,
                                                int64_t part0, float* lds) {
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
      const T* k = reinterpret_cast<const T*>(
          a.k + kvh * a.kh + (uint64_t)((uint32_t)page * a.kp + in * a.ks) * 16) + c * 8;
      const T* v = reinterpret_cast<const T*>(
          a.v + kvh * a.vh + (uint64_t)((uint32_t)page * a.vp + in * a.vs) * 16) + c * 8;
      float x = 0.0f;
      if (on)
        for (int e = 0; e < 8; ++e) x = fmaf(qf[e], io_traits<T>::load(k + e), x);
      for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
      x *= a.scale;
      const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.0f : mn;
      const float was = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(x - base);
      l = fmaf(l, was, p);
      m = mn;
      if (on)
        for (int e = 0; e < 8; ++e) o[e] = fmaf(p, io_traits<T>::load(v + e), o[e] * was);
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
      if (d0 == 0) part_ml(a)[at] = make_float2(mx, sum);
    } else {
      char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                     : b * a.os[0] + t * a.os[1]) + h * a.os[2];
#pragma unroll
      for (int e = 0, d = d0; d < 128; ++e, d += THREADS)
        if (d < a.D)
          io_traits<T>::store(reinterpret_cast<T*>(out) + d, sum == 0.0f ? 0.0f : acc[e] / sum);
      if (d0 == 0 && a.lse != nullptr)
        a.lse[trow * a.NH + h] = sum == 0.0f ? -INFINITY
                                             : (mx + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

template <typename T, int DP, bool PAD, bool FEW>
__global__ void __launch_bounds__((AttnShape<T, FEW>::kThreads), FEW ? 1 : 2)
    attn_tile_kernel(const AttnArgs a) {
  using Ty = AttnType<T>;
  using Ti = AttnTile<T, DP, FEW>;
  using Shape = AttnShape<T, FEW>;
  constexpr int kAttnWaves = Shape::kWaves, kAttnThreads = Shape::kThreads,
                kAttnRows = Shape::kRows;
  constexpr int KT = Ti::kKeys, KB = KT / 32;
  constexpr int kSteps = Ti::kChunks / 2;  // score products' steps: two chunks each
  constexpr int kDB = DP / 32;
  constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;  // a full tile's keys
  constexpr int kRow = Ti::kChunks * 16, kTile = Ti::kUnits * 16;  // bytes
  __shared__ uint4 lds[4 * Ti::kUnits];                            // K, V, and again

  // The lengths of all sequences, a run of them to each thread, and their sum.
  __shared__ uint32_t sums[kAttnWaves];
  __shared__ struct { PagedSeq s; int b; uint32_t at; } found;  // the sequence of a range's begin
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (a.batch.B + kAttnThreads - 1) / kAttnThreads;
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
  for (int w = 0; w < kAttnWaves; ++w) {
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
  const bool full = a.log_group > 0 && line.count << a.log_group == Shape::kGrid;
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
  const int chunks = a.D / Ty::kChunk;

  // Keys begin .. end of a row tile, into its rows of the output or the partials from part0
  // on (-1: none).
  auto piece = [&](int kvh, int tile, int begin, int end, int64_t part0) {
    const char* kbase = a.k + (int64_t)kvh * a.kh;
    const char* vbase = a.v + (int64_t)kvh * a.vh;
    // The page of the lane-th key of a tile, -1: none.
    auto page_of = [&](int kt) {
      const int col = a.batch.div.quot(kt + ((int)threadIdx.x & (KT - 1)));
      const int p = s.table[min(col, a.batch.W - 1)];
      return p < a.batch.P ? p : -1;
    };
    // (opaque: what follows from the lane is not kept in registers around the pieces)
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, ln = lane & 31, hf = lane >> 5;
    uint64_t held = 0;
    // A full tile of pages that all hold keys, and whose sizes are multiples of 16: the
    // rows that a wavefront's load fetches are in one block of kBlock rows and so in one
    // page, and the address is scalar but for an offset that does not change (float32 at
    // 128 channels, whose loads are 8 rows: but for the swizzle of odd ones).
    constexpr int kRows = kAttnThreads / Ti::kChunks, kBlock = kRows < 16 ? kRows : 16;
    const int r0 = (thread / Ti::kChunks) % kBlock, p0 = thread % Ti::kChunks;
    uint32_t koff[16 / kBlock];
#pragma unroll
    for (int x = 0; x < 16 / kBlock; ++x)
      koff[x] = (r0 * a.ks + (p0 ^ Ti::k_swizzle(x * kBlock + r0))) * 16;
    const uint32_t voff = (r0 * a.vs + (p0 ^ Ti::v_swizzle(r0))) * 16;
    static_assert(sizeof(T) == 2 || Ti::kChunks < 32 || kBlock == 8, "V's swizzle repeats in 8 rows");
    // Load x of such a tile: K's and V's alternate.  They are issued between the products of
    // the tile before, as fast as the memory pipe takes them: all at once, each wavefront
    // stands until the others' are through.
    auto load_full = [&](int x, int kt, int page, int buf) {
      const int i = x / 2;
      const bool of_v = x & 1;
      const int r = (i * kRows + wave * (64 / Ti::kChunks)) & ~(kBlock - 1);
      // (without a branch: beside one what is written between the products does not stay there)
      const int j = kt + r;
      const uint32_t from = (uint32_t)__builtin_amdgcn_readlane(page, r);
      const uint32_t at = (uint32_t)(j - a.batch.div.quot_of_many(j) * a.batch.div.size);
      uint4* to = lds + buf * 2 * Ti::kUnits + i * kAttnThreads + wave * 64;
      if (of_v)
        load_lds16(to + Ti::kUnits, vbase + (uint64_t)(from * a.vp + at * a.vs) * 16, voff);
      else
        load_lds16(to, kbase + (uint64_t)(from * a.kp + at * a.ks) * 16, koff[i % (16 / kBlock)]);
    };
    constexpr int kFullLoads = 2 * Ti::kLoads;
    // Whether a tile is one for load_full, and the keys that are there.
    auto is_full = [&](int kt, int page, uint64_t& there) {
      there = __ballot(page >= 0 && kt + (lane & (KT - 1)) < end);
      if constexpr (KT == 32) there &= 0xffffffffull;
      return !PAD && a.scalar_pages && there == kAll;
    };
    // Starts any tile's way into LDS: a thread's chunk u of the buffer is fetched from
    // wherever the swizzle puts it, channels past D are zeros.  For a key past the end the
    // last one is fetched, for one of no page some row: their scores are masked.
    auto load = [&](int kt, int page, int buf) {
      const int j = kt + (lane & (KT - 1)), jj = min(j, end - 1);
      const uint32_t at = (uint32_t)(jj - a.batch.div.quot(jj) * a.batch.div.size);
      const int own = max(page, 0), of_last = __shfl(own, min(lane & (KT - 1), end - 1 - kt));
      const uint32_t from = (uint32_t)(j < end ? own : of_last);
      const uint32_t ku = from * a.kp + at * a.ks;
      const uint32_t vu = from * a.vp + at * a.vs;
      uint32_t kq[Ti::kLoads], vq[Ti::kLoads];
#pragma unroll
      for (int i = 0; i < Ti::kLoads; ++i) {
        const int r = (i * kAttnThreads + thread) / Ti::kChunks;
        kq[i] = __shfl(ku, r);
        vq[i] = __shfl(vu, r);
      }
      in_order();
#pragma unroll
      for (int i = 0; i < Ti::kLoads; ++i) {
        const int u = i * kAttnThreads + thread;
        const int r = u / Ti::kChunks, p = u % Ti::kChunks;
        const int kc = p ^ Ti::k_swizzle(r), vc = p ^ Ti::v_swizzle(r);
        const char* kf = kbase + ((uint64_t)kq[i] + kc) * 16;
        const char* vf = vbase + ((uint64_t)vq[i] + vc) * 16;
        if constexpr (PAD) {
          kf = kc < chunks ? kf : reinterpret_cast<const char*>(&kZeros);
          vf = vc < chunks ? vf : reinterpret_cast<const char*>(&kZeros);
        }
        uint4* to = lds + buf * 2 * Ti::kUnits + i * kAttnThreads + wave * 64;
        load_lds16(to, kf);
        load_lds16(to + Ti::kUnits, vf);
      }
    };

    // Where the lane reads K's row ln, and V's four rows from 4 hf (bfloat16) or row 4 hf
    // (float32), in the first buffer.  The swizzles exclusive-or a slot, so a later step's
    // chunk is an exclusive or away; rows further on a constant.
    const uint32_t lds0 = lds_address(lds);
    const uint32_t kat = lds0 + ln * kRow + (hf ^ Ti::k_swizzle(ln)) * 16;
    uint32_t vat = lds0 + kTile;
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * hf + (lane & 15) / 4;
      vat += r * kRow + ((((lane >> 4) & 1) * 2 + (lane & 3) / 2) ^ Ti::v_swizzle(r)) * 16 +
             (lane & 1) * 8;
    } else {
      vat += 4 * hf * kRow + ((ln / 4) ^ Ti::v_swizzle(4 * hf)) * 16 + (ln % 4) * 4;
    }
    // the first tile on its way before all else
    uint64_t next = 0;
    int page = -1;
    if (begin < end) {
      page = page_of(begin);
      barrier();  // (the row tile before is read to its end)
      is_full(begin, page, next);
      load(begin, page, 0);
      page = page_of(begin + KT);
    }

    // (Of few rows one wavefront has all products: not on the same SIMD in both workgroups of a
    // compute unit.  512 sequences of 100 to 300 tokens 113 us, so and with all wavefronts
    // looking for infinities 109.)
    const int wrow = tile * kAttnRows +
                     (FEW ? 0 : (wave + blockIdx.x / (Shape::kGrid / 2) * 2) & 3) * 32;
    const int rows = s.n * a.g, row = wrow + ln;
    const bool row_ok = row < rows;
    const int t = row_ok ? a.by_g.quot(row) : 0;
    const int h = kvh * a.g + (row_ok ? row - t * a.g : 0);
    const int pos = row_ok ? s.len - s.n + t : -1;
    const int64_t trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;

    // the last position that any row of the wavefront, and of the workgroup, sees
    const bool wave_on = wrow < rows;
    const int wave_end = wave_on ? s.len - s.n + a.by_g.quot(min(wrow + 31, rows - 1)) + 1 : 0;
    const int wave_min = wave_on ? s.len - s.n + a.by_g.quot(wrow) : 0;

    const int first_pos = s.len - s.n + a.by_g.quot(tile * kAttnRows);  // of the tile's rows

    // Q: chunk 2 step + half of the lane's row
    uint4 qf[kSteps];
    {
      const char* q = a.q + (a.batch.starts != nullptr ? trow * a.qs[1]
                                                       : b * a.qs[0] + t * a.qs[1]) + h * a.qs[2];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) qf[i] = make_uint4(0, 0, 0, 0);
      if (row_ok && a.q_aligned) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          if (!PAD || 2 * i + hf < chunks)
            qf[i] = *reinterpret_cast<const uint4*>(q + (2 * i + hf) * 16);
      } else if (row_ok) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int c = 2 * i + hf;
          if (c >= chunks) continue;
          T e[Ty::kChunk];
#pragma unroll
          for (int x = 0; x < Ty::kChunk; ++x)
            e[x] = reinterpret_cast<const T*>(q)[c * Ty::kChunk + x];
          __builtin_memcpy(&qf[i], e, 16);
        }
      }
    }

    f32x16 o[kDB];
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys

    int again = 0;
    if (begin < end) {
      int buf = 0;
      for (int kt = begin; kt < end; kt += KT, buf ^= 1) {
        held = next;
        // every wavefront's loads of this tile have landed, and the other buffer is read
        wait_vmcnt<0>();
        barrier();
        bool full = false;
        const int page_next = page;
        if (kt + KT < end) {
          full = is_full(kt + KT, page, next);
          if (!full) load(kt + KT, page, buf ^ 1);
          page = page_of(kt + 2 * KT);
        }
        if (full && kt >= wave_end) {
#pragma unroll
          for (int x = 0; x < kFullLoads; ++x) load_full(x, kt + KT, page_next, buf ^ 1);
        }
        // A value that some row of the tile may not see must not reach it, not even as 0 times
        // infinity: rows of a masked tile that holds infinities or NaNs are computed again
        // below.  (All wavefronts look, also those without rows.)
        if (held != kAll || kt + KT - 1 > first_pos) {
          bool bad = false;
#pragma unroll
          for (int u = 0; u < Ti::kLoads; ++u)
            bad |= any_nonfinite(lds[(2 * buf + 1) * Ti::kUnits + u * kAttnThreads + thread], T());
          if (__any(bad)) again = 1;
        }
        if (kt < wave_end) {
          const uint32_t ka = kat + buf * 2 * kTile, va = vat + buf * 2 * kTile;
          f32x16 sc[KB];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
          auto scores = [&](auto with_loads) {
            constexpr int N = kSteps * KB, AHEAD = 6;
            u32x4_t kf[AHEAD];
            auto key = [&](int n) {
              return lds_read<u32x4_t>((ka ^ (32 * (n / KB))) + n % KB * 32 * kRow);
            };
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) kf[n] = key(n);
            in_order();
#pragma unroll
            for (int n = 0; n < N; ++n) {
              sc[n % KB] = Ty::scores(kf[n % AHEAD], qf[n / KB], sc[n % KB]);
              if (n + AHEAD < N) kf[n % AHEAD] = key(n + AHEAD);
              if constexpr (decltype(with_loads)::value)
#pragma unroll
                for (int x = n * kFullLoads / N; x < (n + 1) * kFullLoads / N; ++x)
                  load_full(x, kt + KT, page_next, buf ^ 1);
              in_order();
            }
          };
          if (full) scores(std::true_type()); else scores(std::false_type());
          // keys that the lane's row sees, as bits from the lane half's first
          const bool masked = held != kAll || kt + KT - 1 > wave_min;
          uint64_t seen = kAll;
          if (masked) {
            const int n = pos - kt + 1;  // keys up to the row's own
            seen = n <= 0 ? 0 : held & (n >= 64 ? ~0ull : (1ull << n) - 1);
            const uint64_t mine = seen >> (4 * hf);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (!((mine >> (kb * 32 + 8 * (i / 4) + i % 4)) & 1)) sc[kb][i] = -INFINITY;
          }
          float part_top[KB * 2], top = -INFINITY;  // of the lane's keys of each 16
#pragma unroll
          for (int e = 0; e < KB * 2; ++e) {
            part_top[e] = sc[e / 2][8 * (e % 2)];
#pragma unroll
            for (int i = 1; i < 8; ++i) part_top[e] = fmaxf(part_top[e], sc[e / 2][8 * (e % 2) + i]);
            top = fmaxf(top, part_top[e]);
          }
          top = across_halves_max(top) * a.scale;
          // the maximum in use stays until a score passes it by a factor of 2^8: the
          // probabilities stay below 2^8, their sums far from overflow
          if (__any(top > m + 8.0f)) {
            const float mn = fmaxf(m, top);
            // (from here on the argument of an exponential, a fused multiply and subtract of
            // a rounded product, is off by 2^-6 and more: one by one it never exceeds 0)
            if (__any(fabsf(mn) > 0x1p18f && mn != -INFINITY)) again = 1;
            const float was = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= was;
#pragma unroll
            for (int d = 0; d < kDB; ++d)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[d][i] *= was;
          }
          const float base = m == -INFINITY ? 0.0f : m;
          auto prob = [&](int kb, int i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], a.scale, -base));
            sc[kb][i] = p;
            l += p;
          };
          // O^T += V^T P^T
          if constexpr (sizeof(T) == 2) {
            constexpr int N = KB * 2;  // steps of 16 keys
            uint4 vf[2][kDB];
            auto value = [&](int e, int d) {
              typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
              union {
                s16x4 half[2];
                uint4 v;
              } f;
#pragma unroll
              for (int x = 0; x < 2; ++x)
                f.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4*)(uintptr_t)((va ^ (64 * d)) + (16 * e + 8 * x) * kRow));
              return f.v;
            };
            auto product = [&](int d, uint4 v, uint4 p) {
              o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  __builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, p), o[d], 0, 0, 0);
            };
            // probabilities 2 x, 2 x + 1 of step e
            auto pair = [&](int e, int x) {
              const int i = 8 * (e % 2) + 2 * x;
              prob(e / 2, i);
              prob(e / 2, i + 1);
              return cvt_pk_bf16(sc[e / 2][i], sc[e / 2][i + 1]);
            };
            // A probability is rounded to bfloat16 for the product, by 2^-8 of it at most, and
            // what is left of it is multiplied too: the outputs then are off by their own
            // rounding only.  Where the products bound a call (plan_shape) that is done for 16
            // keys with one that weighs more than about a 32nd of its row so far; of the
            // others' errors, each as large as the output's rounding beside its own term, part
            // stays: 12,289 tokens over 32,289 have a relative error (of the whole output, of
            // values around 0) of 0.00193 in place of 0.00166, and take 1,157 us in place of
            // 1,427.
            uint32_t fine = a.all_rests ? (1u << N) - 1 : 0;
            if (!a.all_rests && __any(__builtin_amdgcn_exp2f(top - base) * 16.0f > l)) {
#pragma unroll
              for (int e = 0; e < N; ++e)
                if (__any(__builtin_amdgcn_exp2f(fmaf(part_top[e], a.scale, -base)) * 16.0f > l))
                  fine |= 1u << e;
            }
            uint32_t w[4], next[4];
#pragma unroll
            for (int d = 0; d < kDB; ++d) vf[0][d] = value(0, d);
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = pair(0, x);
            in_order();
#pragma unroll
            for (int e = 0; e < N; ++e) {
#pragma unroll
              for (int d = 0; d < kDB; ++d) {
                product(d, vf[e & 1][d], make_uint4(w[0], w[1], w[2], w[3]));
                if (e + 1 < N) {
                  vf[(e + 1) & 1][d] = value(e + 1, d);
#pragma unroll
                  for (int x = d * 4 / kDB; x < (d + 1) * 4 / kDB; ++x) next[x] = pair(e + 1, x);
                }
                in_order();
              }
              if (fine & (1u << e)) {
                uint32_t rest[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const int i = 8 * (e % 2) + 2 * x;
                  rest[x] = cvt_pk_bf16(sc[e / 2][i] - __uint_as_float(w[x] << 16),
                                        sc[e / 2][i + 1] - __uint_as_float(w[x] & 0xffff0000u));
                }
#pragma unroll
                for (int d = 0; d < kDB; ++d)
                  product(d, vf[e & 1][d], make_uint4(rest[0], rest[1], rest[2], rest[3]));
              }
#pragma unroll
              for (int x = 0; x < 4; ++x) w[x] = next[x];
            }
          } else {
            constexpr int N = 16 * kDB, AHEAD = 8;
            float vf[AHEAD];
            auto value = [&](int n) {
              const int i = n / kDB;
              return lds_read<float>((va ^ (128 * (n % kDB))) + (8 * (i / 4) + i % 4) * kRow);
            };
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) vf[n] = value(n);
            prob(0, 0);
            prob(0, 1);
            in_order();
#pragma unroll
            for (int n = 0; n < N; ++n) {
              o[n % kDB] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[n % AHEAD], sc[0][n / kDB],
                                                                o[n % kDB], 0, 0, 0);
              if (n + AHEAD < N) vf[n % AHEAD] = value(n + AHEAD);
              if (n % kDB == 0 && n / kDB + 2 < 16) prob(0, n / kDB + 2);
              in_order();
            }
          }
        }
      }
    }

    if (__syncthreads_or(again)) {
      rows_one_by_one<T, kAttnThreads>(a, s, b, kvh, tile * kAttnRows, min(rows, (tile + 1) * kAttnRows), begin,
                         end, part0, reinterpret_cast<float*>(lds));
      return;
    }
    l += __shfl_xor(l, 32);
    if (row_ok) {
      if (part0 >= 0) {
        const int64_t at = part0 + row - tile * kAttnRows;
        float* po = a.part + at * a.D;
#pragma unroll
        for (int d = 0; d < kDB; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int ch = d * 32 + 2 * i + 4 * hf;
            if (ch < a.D)
              *reinterpret_cast<float4*>(po + ch) =
                  make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
          }
        if (hf == 0) part_ml(a)[at] = make_float2(m, l);
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                       : b * a.os[0] + t * a.os[1]) + h * a.os[2];
#pragma unroll
        for (int d = 0; d < kDB; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int ch = d * 32 + 2 * i + 4 * hf;
            if (ch >= a.D) continue;
            const float x[4] = {o[d][i] * inv, o[d][i + 1] * inv, o[d][i + 2] * inv,
                                o[d][i + 3] * inv};
            if constexpr (sizeof(T) == 2)
              *reinterpret_cast<uint2*>(out + ch * 2) =
                  make_uint2(cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]));
            else
              *reinterpret_cast<float4*>(out + ch * 4) = make_float4(x[0], x[1], x[2], x[3]);
          }
        if (hf == 0 && a.lse != nullptr)
          a.lse[trow * a.NH + h] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
      }
    }
  };

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
    const bool cuts = min(rows, kAttnRows) <= a.part_tile;
    if (on && (cuts || from == 0)) {
      const bool whole = !cuts || (from == 0 && to == c);
      const int keys = keys_of(a, s, tile), blocks = (keys + KT - 1) / KT;
      const int begin = whole ? 0 : cut_at(from, c, blocks, a.extra) * KT;
      const int end = whole || to == c ? keys : min(keys, cut_at(to, c, blocks, a.extra) * KT);
      if (x == x0 && from > 0 && at >= line.begin(range - 1) && threadIdx.x == 0)
        a.cuts[(range << a.log_group) + member] =
            Cut{min(rows - tile * kAttnRows, kAttnRows), b, kvh, (int)s.row0, tile,
                line.of(at + c - 1), {}};
      if (!whole && begin >= end) {  // (a piece of no keys)
        const int64_t part0 = part_at(a, range, member, from == 0);
        if ((int)threadIdx.x < min(rows - tile * kAttnRows, kAttnRows))
          part_ml(a)[part0 + threadIdx.x] = make_float2(-INFINITY, 0.0f);
      } else {
        piece(kvh, tile, begin, end, whole ? -1 : part_at(a, range, member, from == 0));
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

template <typename T, bool FEW>
AttnPlan plan_shape(const ltv_paged_batch& b, int NH, int NKVH, int D, int max_len) {
  using Shape = AttnShape<T, FEW>;
  constexpr int KT = Shape::kKeys, kAttnRows = Shape::kRows;
  AttnPlan p;
  p.few = FEW;
  p.log_rows = FEW ? 5 : 7;
  const int64_t g = NH / NKVH, rows = std::max(b.T, 1) * g;
  const int64_t tiles = (rows + kAttnRows - 1) / kAttnRows;
  // Groups of four (one, two and four: 132, 126 and 112 us of chunks among decoding sequences,
  // 1,270, 1,246 and 1,239 of the long prompt); float32, whose products take eight times as
  // long as its reads, is better off with each tile by itself (one and four: 49.6 and 52.2).
  p.group = FEW || sizeof(T) == 4 ? 1 : tiles >= 3 ? 4 : (int)tiles;
  p.group_tokens = (int)((p.group * kAttnRows + g - 1) / g);
  // (where no sequence can have more than a block of keys none is cut)
  const int64_t keys = (int64_t)b.table_width * b.page_size;
  p.joins = keys > KT;
  p.part_tile = p.joins ? (int)std::min<int64_t>(rows, kAttnRows) : 0;
  // (of few rows all their latency is a tile's: there no range is too short, 18.5 us of a small
  // decode step and 20.9 with two)
  p.least = (rows <= 32 ? 64 : 128) / KT;
  // (fewer, if the call has no more tiles than that)
  const int64_t groups =
      NKVH * std::min((tiles + p.group - 1) / p.group * b.B,
                      b.total * g / (p.group * kAttnRows) + b.B);
  const int64_t most = groups * ((std::max(max_len, 1) + KT - 1) / KT);
  p.ranges = (int)std::min<int64_t>(Shape::kGrid / p.group, (most + p.least - 1) / p.least);
  p.ranges = std::max(8, (p.ranges + 7) / 8 * 8);
  // Positions on the line have 32 bits: units of more blocks where it could be longer than
  // 2^30, whatever the lengths are.
  const double bound = (double)NKVH * ((double)b.total * g / (p.group * kAttnRows) + b.B) *
                       ((double)(keys + b.total) / KT + 64);
  p.unit = 0;
  while (bound / (double)(int64_t(1) << p.unit) > (double)(1 << 30)) ++p.unit;
  p.slope = (int)(p.group * kAttnRows / g / KT) >> p.unit;
  // What a piece costs beside its keys -- its rows, the first tile's way, the remainders that
  // the first tiles take, its partials -- counted in blocks: four, or none where few rows have
  // a range for every few blocks.  (Without and with it: chunks mixed with decoding 110 and 98
  // us, float32 chunks 50 and 48, a ragged decode step 282 and 261; a small one 17.6 and, with
  // one block, 18.4.  Two, four and eight for 256 sequences of up to 2,000 tokens 222, 219, 224.)
  p.extra = (FEW || rows > 32 || most > 8 * Shape::kGrid ? 4 : 0) >> p.unit;
  // Up to 10^11 operations, by the hints, the products of all probabilities' rests cost next to
  // nothing: 64 sequences of 8,000 tokens (4 heads) 183 us without most of them and 185 with all,
  // 128 of up to 2,000 (8 heads) 108 and 111, 64 of 8,000 with 64 channels (8 heads) 213 and 222,
  // 1,024 new tokens over 8,000 (6 heads) 68.6 and 67.5.  Beyond, 2,048 over 16,000 take 178 and
  // 183, 4,096 over 32,000 518 and 618.
  p.all_rests = 4.0 * D * NH * (double)b.total * std::max(max_len, 1) <= 1e11;
  const int64_t n = (int64_t)p.ranges * p.group;
  p.part_rows = n * 2 * p.part_tile;
  p.cuts_at = (size_t)p.part_rows * (D + 2) * sizeof(float);
  p.bytes = p.cuts_at + n * sizeof(Cut) + 16;
  return p;
}

// Which shape.  One wavefront in four workgroups of a unit where there are many sequences of few
// rows that are not long: a step of 2,048 sequences of 30 to 100 tokens (6 heads) 246 us with
// four wavefronts and 167 with one, 512 of 100 to 300 99 and 82, 32 of 300 to 700 26.4 and 21.9,
// 40 of 200 to 1,000 (8 heads) 29.3 and 29.1.  Of long ones the pieces are more to join and the
// tiles half as large: 128 of up to 2,000 (8 heads) 119 and 123, 64 of 8,000 (4 heads) 183 and
// 187.  Where there are very many the longest says little about the others, and one wavefront
// has less to lose: 256 of up to 2,000 (8 heads) 213 and 219.  With little work what counts is
// how soon a tile is there, which four wavefronts load together (four sequences 17.9 and 23.0);
// of more rows, too, the pieces weigh more (32 rows 46.5 and 49.2).  float32 has its products
// to wait for.
AttnPlan plan_attention(const ltv_paged_batch& b, int dtype, int NH, int NKVH, int D, int max_len) {
  if (dtype == LTV_DTYPE_F32) return plan_shape<float, false>(b, NH, NKVH, D, max_len);
  const int64_t rows = (int64_t)std::max(b.T, 1) * (NH / NKVH), units = (int64_t)b.B * NKVH;
  const int64_t blocks = units * ((std::max(max_len, 1) + 63) / 64);
  if (rows <= 16 && blocks >= 1024 && (max_len <= 1024 || units >= 2048))
    return plan_shape<bf16_t, true>(b, NH, NKVH, D, max_len);
  return plan_shape<bf16_t, false>(b, NH, NKVH, D, max_len);
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_paged_attention_workspace_size(int dtype, const ltv_paged_batch* batch,
                                                     int NH, int NKVH, int D, int max_len) {
  if (batch == nullptr || batch->B <= 0 || batch->T < 0 || NKVH <= 0 || NH < NKVH || D <= 0)
    return 0;
  return plan_attention(*batch, dtype, NH, NKVH, D, max_len).bytes;
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
  LTV_REQUIRE(scale > 0.0f && scale * kLog2e < INFINITY, LTV_ERR_INVALID_ARG,
              "scale must be positive and finite (%g)", scale);
  if (batch->B == 0 || batch->total == 0 || NH == 0) return LTV_OK;
  LTV_REQUIRE(batch->total * NH < (int64_t(1) << 30), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  const bool pages = batch->num_pages > 0;
  LTV_REQUIRE(q && out && q_strides && out_strides && k_page_strides && v_page_strides &&
                  (!pages || (k_pages && v_pages)),
              LTV_ERR_INVALID_ARG, "null pointer");
  const int es = elem_size(dtype), chunk = 16 / es;
  const AttnPlan p = plan_attention(*batch, dtype, NH, NKVH, D, max_len);
  LTV_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= p.bytes, LTV_ERR_WORKSPACE,
              "workspace too small");
  // pages are addressed in 16-byte units of 32 bits
  bool fits = true, aligned = aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 3; ++i)
    for (const int64_t st : {k_page_strides[i], v_page_strides[i]}) {
      aligned = aligned && st % chunk == 0;
      const int64_t n = i == 0 ? batch->num_pages : i == 1 ? 1 : batch->page_size;
      fits = fits && st >= 0 && (st == 0 || n <= (int64_t(1) << 31) / std::max<int64_t>(1, st / chunk));
    }
  // (16 rows' offsets in 32 bits)
  const bool rows_fit = k_page_strides[2] < (1 << 20) && v_page_strides[2] < (1 << 20);
  LTV_REQUIRE(!pages || aligned, LTV_ERR_UNSUPPORTED, "the pages' rows must be 16-byte aligned");
  LTV_REQUIRE(!pages || fits, LTV_ERR_UNSUPPORTED,
              "the pages of a layer must lie within 32 GiB, with strides that are not negative");
  bool out_ok = aligned16(out), q_aligned = aligned16(q);
  for (int i = batch->starts != nullptr ? 1 : 0; i < 3; ++i) {
    out_ok = out_ok && out_strides[i] % chunk == 0;
    q_aligned = q_aligned && q_strides[i] % chunk == 0;
  }
  LTV_REQUIRE(out_ok, LTV_ERR_UNSUPPORTED, "the output's rows must be 16-byte aligned");
  AttnArgs a{PagedBatch(*batch), (const char*)q, (const char*)k_pages, (const char*)v_pages,
             (char*)out, lse, (float*)workspace, {}, {}, k_page_strides[1] * es,
             v_page_strides[1] * es, (uint32_t)(k_page_strides[0] / chunk),
             (uint32_t)(k_page_strides[2] / chunk), (uint32_t)(v_page_strides[0] / chunk),
             (uint32_t)(v_page_strides[2] / chunk), NH, NKVH, D, NH / NKVH, q_aligned ? 1 : 0, p.all_rests ? 1 : 0,
             rows_fit && batch->page_size % 16 == 0,
             scale * kLog2e, p.group == 4 ? 2 : p.group - 1, p.ranges, p.least, p.unit,
             p.group_tokens, p.slope, p.extra, p.log_rows, p.part_tile, PageDiv(NH / NKVH),
             PageDiv(p.ranges), p.part_rows, nullptr, nullptr};
  a.cuts = (Cut*)((char*)workspace + p.cuts_at);
  a.head = (int*)(a.cuts + (size_t)p.ranges * p.group);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i] * es;
    a.os[i] = out_strides[i] * es;
  }
  const unsigned grid = p.ranges * p.group;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, st, a);
  };
  auto by_width = [&](auto type, auto few) {
    using T = decltype(type);
    constexpr bool F = decltype(few)::value;
    constexpr int threads = AttnShape<T, F>::kThreads;
    if (D == 64) launch(attn_tile_kernel<T, 64, false, F>, threads);
    else if (D < 64) launch(attn_tile_kernel<T, 64, true, F>, threads);
    else if (D == 128) launch(attn_tile_kernel<T, 128, false, F>, threads);
    else launch(attn_tile_kernel<T, 128, true, F>, threads);
  };
  if (dtype == LTV_DTYPE_F32) by_width(float(), std::false_type());
  else if (p.few) by_width(bf16_t(), std::true_type());
  else by_width(bf16_t(), std::false_type());
  LTV_LAUNCH_CHECK();
  if (p.joins) {
    auto join = [&](auto type) {
      using T = decltype(type);
      const int each = p.part_tile <= 16 ? 1 : 8;
      hipLaunchKernelGGL(attn_join_kernel<T>, dim3(grid, (p.part_tile + each - 1) / each),
                         dim3(256), 0, st, a, each);
    };
    if (dtype == LTV_DTYPE_F32) join(float()); else join(bf16_t());
    LTV_LAUNCH_CHECK();
  }
  return LTV_OK;
}
