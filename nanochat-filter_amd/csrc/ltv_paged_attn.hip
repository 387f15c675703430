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
// reads its keys once.  A workgroup has 128 rows, 32 for each of four wavefronts.
//
// Layout of the products (32 x 32 MFMA blocks).  The scores are computed as S^T = K Q^T:
// a lane then holds 16 keys of one row, so maximum and sum are taken in the lane and
// once across the two half-wavefronts, and its values are, without any exchange, the
// right-hand operand of O^T = V^T P^T: the order of the keys within a product is free
// as long as V^T is read in the same one (ds_read_b64_tr_b16 transposes four keys of a
// column at a time).  Both tiles are shared by the wavefronts through LDS, two buffers
// deep: the next tile is on its way, straight into LDS, while this one is computed.
//
// Split.  Few rows and many keys leave compute units idle, so a sequence's keys are cut
// into chunks that workgroups take side by side; a second kernel joins their (m, l, o).
#include <algorithm>
#include <type_traits>

#include "ltv_gemm_dma.hpp"
#include "ltv_paged.hpp"

namespace ltv {
namespace {

constexpr int kAttnWaves = 4;
constexpr int kAttnThreads = kAttnWaves * 64;
constexpr int kAttnRows = kAttnWaves * 32;  // rows of a workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  PagedBatch batch;
  const char* q;
  const char* k;
  const char* v;
  char* out;
  float* lse;
  float* part;                // partial o, then (m, l), of the split sequences
  int64_t qs[3], os[3];       // bytes
  int64_t kh, vh;             // bytes from head to head of the pages
  uint32_t kp, ks, vp, vs;    // 16-byte units from page to page and row to row
  int NH, NKVH, D, g;
  int q_aligned;
  int scalar_pages;           // load_full: 1 pages are multiples of 16 rows, 2 of 64
  float scale;                // with log2(e)
  int tiles, group;           // row tiles of the grid, and how many follow each other
  int chunk, nsplit;          // keys of a split, splits of the grid
  int64_t rows_cap;           // sequences of more rows are not split
  int by_token;               // how the partials are laid out
  int64_t part_rows;
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
  static constexpr int kKeys = 64;  // keys of a tile
  // S^T += K Q^T over 16 channels: a lane's k and q chunk hold channels 8 (lane / 32) ..
  static __device__ __forceinline__ f32x16 scores(u32x4_t k, uint4 q, f32x16 s) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                   __builtin_bit_cast(bf16x8_t, q), s, 0, 0, 0);
  }
};

template <>
struct AttnType<float> {
  static constexpr int kChunk = 4;
  static constexpr int kKeys = 32;
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
template <typename T, int DP>
struct AttnTile {
  static constexpr int kKeys = AttnType<T>::kKeys;
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

// (row numbers stay below 2^30: divisions of 64 bits would take longer than small calls)
__device__ __forceinline__ int over(int a, int b) { return (int)((unsigned)a / (unsigned)b); }

// The splits of a sequence: 1, or how many chunks its keys make.
__device__ __forceinline__ int splits_of(const AttnArgs& a, const PagedSeq& s) {
  if ((int64_t)s.n * a.g > a.rows_cap) return 1;
  return max(1, min(a.nsplit, (s.len + a.chunk - 1) / a.chunk));
}

// A row's place among the partials (D values each; behind them all, its m and l): by its
// token and head where any sequence may be split, else among the rows_cap of its sequence
// and k/v head.
__device__ __forceinline__ int64_t part_row(const AttnArgs& a, int bh, int split, int64_t row,
                                            int64_t trow, int h) {
  if (a.by_token) return ((int64_t)split * a.batch.total + trow) * a.NH + h;
  return ((int64_t)bh * a.nsplit + split) * a.rows_cap + row;
}
__device__ __forceinline__ float2* part_ml(const AttnArgs& a) {
  return reinterpret_cast<float2*>(a.part + a.part_rows * a.D);
}

// Rows row0 .. row_end - 1 of a workgroup over keys begin .. end - 1, each key that a row
// does not see left alone altogether: the way of tiles with infinite or NaN values among
// those that some rows do not see.  Sixteen groups of sixteen lanes take a row's keys in
// turn, a lane holding eight channels.  split: whose partials these are, or -1.
template <typename T>
__device__ __forceinline__ void rows_one_by_one(const AttnArgs& a, const PagedSeq& s, int b,
                                                int kvh, int row0, int row_end, int begin, int end,
                                                int split, float* lds) {
#pragma clang fp contract(off)  // (x - base below must not be a fused form of the product)
  float* lds_m = lds;
  float* lds_l = lds + 16;
  float* lds_o = lds + 32;  // 16 x 128
  const int c = threadIdx.x & 15, gi = threadIdx.x >> 4;
  const bool on = c * 8 < a.D;
  for (int row = row0; row < row_end; ++row) {
    const int t = over(row, a.g), h = kvh * a.g + row - t * a.g;
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
    for (int j = begin + gi; j <= last; j += 16) {
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
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, lds_m[i]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, acc = 0.0f;
    const int d = threadIdx.x;
    for (int i = 0; i < 16; ++i) {
      // (a group without keys has weight 0)
      const float w = lds_m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lds_m[i] - base);
      sum = fmaf(lds_l[i], w, sum);
      if (d < a.D) acc = fmaf(lds_o[i * 128 + d], w, acc);
    }
    if (split >= 0) {
      const int64_t at = part_row(a, b * a.NKVH + kvh, split, row, trow, h);
      if (d < a.D) a.part[at * a.D + d] = acc;
      if (d == 0) part_ml(a)[at] = make_float2(mx, sum);
    } else {
      char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                     : b * a.os[0] + t * a.os[1]) + h * a.os[2];
      if (d < a.D)
        io_traits<T>::store(reinterpret_cast<T*>(out) + d, sum == 0.0f ? 0.0f : acc / sum);
      if (d == 0 && a.lse != nullptr)
        a.lse[trow * a.NH + h] = sum == 0.0f ? -INFINITY
                                             : (mx + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

template <typename T, int DP, bool PAD>
__global__ void __launch_bounds__(kAttnThreads, 2) attn_tile_kernel(const AttnArgs a) {
  using Ty = AttnType<T>;
  using Ti = AttnTile<T, DP>;
  constexpr int KT = Ti::kKeys, KB = KT / 32;
  constexpr int kSteps = Ti::kChunks / 2;  // score products' steps: two chunks each
  constexpr int kDB = DP / 32;
  constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;  // a full tile's keys
  constexpr int kRow = Ti::kChunks * 16, kTile = Ti::kUnits * 16;  // bytes
  __shared__ uint4 lds[4 * Ti::kUnits];                            // K, V, and again

  // Workgroup w runs on XCD w % 8.  Up to four row tiles that read the same keys -- those of
  // one sequence, k/v head and split -- follow each other on one XCD, whose L2 then holds
  // the keys for all but the first of them; such groups go around the XCDs, those of the
  // last rows, with the most keys, first.  A sequence's splits start at an XCD that differs
  // by sequence and head, or those in use of short sequences would land on few of them.
  const int xcd = blockIdx.x & 7, place = blockIdx.x >> 3;
  const int round = over(place, a.group), unit = round * 8 + xcd;
  const int pairs = a.batch.B * a.NKVH * a.nsplit, rank = over(unit, pairs);
  const int pair = unit - rank * pairs, bh = over(pair, a.nsplit);
  const int tile0 = a.tiles - 1 - rank * a.group - (place - round * a.group);
  if (tile0 < 0) return;
  const int split = (int)((unsigned)(pair - bh * a.nsplit + bh) % (unsigned)a.nsplit);
  const int b = over(bh, a.NKVH), kvh = bh - b * a.NKVH;
  const PagedSeq s = paged_seq(a.batch, b);
  // The page of the lane-th key of a tile, -1: none.  (Read without waiting for the
  // sequence's length; what is past the end is sorted out where it is used.)
  auto page_of = [&](int kt) {
    const int col = a.batch.div.quot(kt + ((int)threadIdx.x & (KT - 1)));
    const int p = a.batch.W > 0 ? s.table[min(col, a.batch.W - 1)] : -1;
    return p < a.batch.P ? p : -1;
  };
  const int begin = split * a.chunk, first_page = page_of(begin);
  const int nsplit = splits_of(a, s);
  if (split >= nsplit) return;
  const int rows = s.n * a.g;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const char* kbase = a.k + (int64_t)kvh * a.kh;
  const char* vbase = a.v + (int64_t)kvh * a.vh;
  const int chunks = a.D / Ty::kChunk;

  // (more rows than the grid was sized for: its tiles are walked again)
  for (int tile = tile0; tile * kAttnRows < rows; tile += a.tiles) {
    // (opaque: what follows from the lane is not kept in registers around this loop)
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, ln = lane & 31, hf = lane >> 5;
    const int row = tile * kAttnRows + wave * 32 + ln;
    const bool row_ok = row < rows;
    const int t = row_ok ? over(row, a.g) : 0;
    const int h = kvh * a.g + (row_ok ? row - t * a.g : 0);
    const int pos = row_ok ? s.len - s.n + t : -1;
    const int64_t trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;

    // the last position that any row of the wavefront, and of the workgroup, sees
    const bool wave_on = tile * kAttnRows + wave * 32 < rows;
    const int wfirst = tile * kAttnRows + wave * 32, last = rows - 1;
    const int wave_end = wave_on ? s.len - s.n + over(min(wfirst + 31, last), a.g) + 1 : 0;
    const int wave_min = wave_on ? s.len - s.n + over(wfirst, a.g) : 0;
    const int tlast = over(min(tile * kAttnRows + kAttnRows - 1, last), a.g);
    int end = a.batch.P > 0 ? s.len - s.n + tlast + 1 : 0;
    if (split < nsplit - 1) end = min(end, begin + a.chunk);

    // Q: chunk 2 step + half of the lane's row
    uint4 qf[kSteps];
    {
      const char* q = a.q + (a.batch.starts != nullptr ? trow * a.qs[1]
                                                       : b * a.qs[0] + t * a.qs[1]) + h * a.qs[2];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int c = 2 * i + hf;
        qf[i] = make_uint4(0, 0, 0, 0);
        if (row_ok && c < chunks) {
          if (a.q_aligned) {
            qf[i] = *reinterpret_cast<const uint4*>(q + c * 16);
          } else {
            T e[Ty::kChunk];
#pragma unroll
            for (int x = 0; x < Ty::kChunk; ++x)
              e[x] = reinterpret_cast<const T*>(q)[c * Ty::kChunk + x];
            __builtin_memcpy(&qf[i], e, 16);
          }
        }
      }
    }

    f32x16 o[kDB];
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys

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
      // (pages of whole tiles: one page and row, and constant steps from it)
      const int j = a.scalar_pages == 2 ? kt : kt + r;
      uint32_t at = (uint32_t)(j - a.batch.div.quot(j) * a.batch.div.size);
      const uint32_t from = (uint32_t)__builtin_amdgcn_readlane(page, a.scalar_pages == 2 ? 0 : r);
      if (a.scalar_pages == 2) at += r;
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
    int again = 0;
    if (begin < end) {
      int page = first_page;
      barrier();  // (the row tile before is read to its end)
      uint64_t next;
      is_full(begin, page, next);
      load(begin, page, 0);
      page = page_of(begin + KT);
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
        if (kt < wave_end) {
          const uint32_t ka = kat + buf * 2 * kTile, va = vat + buf * 2 * kTile;
          f32x16 sc[KB];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
          auto scores = [&](auto with_loads) {
            constexpr int N = kSteps * KB, AHEAD = 6;
            static_assert(N == 2 * kFullLoads, "a load to two products");
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
              if (decltype(with_loads)::value && (n & 1))
                load_full(n / 2, kt + KT, page_next, buf ^ 1);
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
          // A value that some row of the tile may not see must not reach it, not even as
          // 0 times infinity: rows of a masked tile that holds infinities or NaNs are
          // computed again below.
          if (masked) {
            bool bad = false;
#pragma unroll 4
            for (int u = lane; u < Ti::kUnits; u += 64) 
              bad |= any_nonfinite(lds[(2 * buf + 1) * Ti::kUnits + u], T());
            if (__any(bad)) again = 1;
          }
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
            // A probability is rounded to bfloat16 for the product, by 2^-8 of it at most.  Of
            // 16 keys with one that weighs more than about a 32nd of its row so far, the rest
            // is multiplied too; below that, the errors of a row's many terms average out far
            // under the output's own rounding.
            uint32_t fine = 0;
            if (__any(__builtin_amdgcn_exp2f(top - base) * 16.0f > l)) {
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
      rows_one_by_one<T>(a, s, b, kvh, tile * kAttnRows, min(rows, (tile + 1) * kAttnRows), begin,
                         end, nsplit > 1 ? split : -1, reinterpret_cast<float*>(lds));
      continue;
    }
    l += __shfl_xor(l, 32);
    if (row_ok) {
      if (nsplit > 1) {
        const int64_t at = part_row(a, bh, split, row, trow, h);
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
  }
}

// Joins the splits of a row: W wavefronts per row take them in turn, a lane two channels
// (one wavefront, four rows to a workgroup, up to 16 splits; else 4 or 16).
template <typename T, int W>
__global__ void __launch_bounds__(W < 4 ? 256 : W * 64) attn_join_kernel(const AttnArgs a) {
  __shared__ float lds_o[W][128];
  __shared__ float lds_l[W];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6;
  int unit = blockIdx.x;
  if (W == 1) unit = unit * 4 + (threadIdx.x >> 6);
  int b, h, row, t;
  int64_t trow;
  PagedSeq s;
  if (a.by_token) {
    const int token = over(unit, a.NH);
    trow = token;
    h = unit - token * a.NH;
    if (trow >= a.batch.total) return;
    if (a.batch.starts != nullptr) {
      // the last sequence that starts at the row or before it
      int lo = 0, hi = a.batch.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.batch.starts[mid] <= trow) lo = mid; else hi = mid - 1;
      }
      b = lo;
    } else {
      b = over(token, a.batch.T);
    }
    s = paged_seq(a.batch, b);
    t = (int)(a.batch.starts != nullptr ? trow - s.row0 : trow - (int64_t)b * a.batch.T);
    if (t < 0 || t >= s.n) return;
    row = t * a.g + h % a.g;
  } else {
    const int nbh = a.batch.B * a.NKVH;
    row = over(unit, nbh);
    const int bh = unit - row * nbh;
    b = over(bh, a.NKVH);
    s = paged_seq(a.batch, b);
    if (row >= a.rows_cap || row >= s.n * a.g) return;
    t = over(row, a.g);
    h = (bh - b * a.NKVH) * a.g + row - t * a.g;
    trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;
  }
  const int nsplit = splits_of(a, s);
  if (nsplit <= 1) return;
  const int bh = b * a.NKVH + over(h, a.g);
  const int64_t first = part_row(a, bh, 0, row, trow, h);
  const int64_t step = part_row(a, bh, 1, row, trow, h) - first;
  const float2* ml = part_ml(a) + first;
  const float* part = a.part + first * a.D;
  float m = -INFINITY;
  for (int i = lane; i < nsplit; i += 64) m = fmaxf(m, ml[i * step].x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float base = m == -INFINITY ? 0.0f : m;
  const bool on = lane * 2 < a.D;
  float ox = 0.0f, oy = 0.0f, l = 0.0f;
#pragma unroll 4
  for (int i = wave; i < nsplit; i += W) {
    const float2 p = ml[i * step];
    const float2 x = on ? *reinterpret_cast<const float2*>(part + i * step * a.D + lane * 2)
                        : make_float2(0.0f, 0.0f);
    // (a split without keys has weight 0; its sums are 0 too)
    const float w = __builtin_amdgcn_exp2f(p.x - base);
    l = fmaf(p.y, w, l);
    ox = fmaf(x.x, w, ox);
    oy = fmaf(x.y, w, oy);
  }
  if constexpr (W > 1) {
    if (on) {
      lds_o[wave][lane * 2] = ox;
      lds_o[wave][lane * 2 + 1] = oy;
    }
    if (lane == 0) lds_l[wave] = l;
    __syncthreads();
    if (wave != 0) return;
    ox = oy = l = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      l += lds_l[w];
      if (on) {
        ox += lds_o[w][lane * 2];
        oy += lds_o[w][lane * 2 + 1];
      }
    }
  }
  char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                 : b * a.os[0] + t * a.os[1]) + h * a.os[2];
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (on) {
    if constexpr (sizeof(T) == 2)
      reinterpret_cast<uint32_t*>(out)[lane] = cvt_pk_bf16(ox * inv, oy * inv);
    else
      reinterpret_cast<float2*>(out)[lane] = make_float2(ox * inv, oy * inv);
  }
  if (lane == 0 && a.lse != nullptr)
    a.lse[trow * a.NH + h] = l == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(l)) * kLn2;
}

// How a call is cut: row tiles of the grid, keys of a split, splits, and where the
// splits' partials go.
struct AttnPlan {
  int tiles, group, chunk, nsplit, by_token;
  int64_t rows_cap, joins, part_rows;
};

AttnPlan plan_attention(const ltv_paged_batch& b, int NH, int NKVH, int max_len) {
  AttnPlan p;
  const int64_t g = NH / NKVH, rows = std::max(b.T, 1) * g, seqs = (int64_t)b.B * NKVH;
  p.tiles = (int)std::min<int64_t>((rows + kAttnRows - 1) / kAttnRows, 1 << 20);
  const int groups = (p.tiles + 3) / 4;
  p.group = (p.tiles + groups - 1) / groups;
  // The row tiles there are at most.  The card holds 512 workgroups at a time (two per
  // compute unit).  With fewer row tiles than five times that, every sequence is split
  // into about that many workgroups, or the last ones of few would run alone; else those
  // of a single tile are.  Chunks of at most 1,024 keys for each tile of a sequence keep
  // a long one from outlasting the others.
  const int64_t tiles = std::min(seqs * p.tiles, (b.total * g / kAttnRows + b.B) * NKVH);
  p.by_token = tiles < 2560;
  p.rows_cap = p.by_token ? int64_t(1) << 40 : std::min<int64_t>(rows, kAttnRows);
  const int64_t keys = std::max(max_len, 1);
  const int64_t want = keys * (p.by_token ? tiles : seqs) / 2560;
  const int64_t least = rows <= 32 ? 64 : 128;  // (of few rows: all their latency is a tile's)
  p.chunk = (int)std::min<int64_t>(std::max<int64_t>((want + 63) / 64 * 64, least),
                                   p.by_token ? int64_t(1024) * p.tiles : 1024);
  p.nsplit = (int)((keys + p.chunk - 1) / p.chunk);
  p.joins = p.by_token ? b.total * NH : seqs * p.rows_cap;
  p.part_rows = p.nsplit * (p.by_token ? b.total * NH : seqs * p.rows_cap);
  return p;
}

size_t part_bytes(const AttnPlan& p, int D) {
  return p.nsplit <= 1 ? 0 : (size_t)p.part_rows * (D + 2) * sizeof(float);
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_paged_attention_workspace_size(int dtype, const ltv_paged_batch* batch,
                                                     int NH, int NKVH, int D, int max_len) {
  if (batch == nullptr || batch->B <= 0 || batch->T < 0 || NKVH <= 0 || NH < NKVH || D <= 0)
    return 0;
  return part_bytes(plan_attention(*batch, NH, NKVH, max_len), D);
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
  LTV_REQUIRE(scale > 0.0f && scale < INFINITY, LTV_ERR_INVALID_ARG,
              "scale must be positive and finite (%g)", scale);
  if (batch->B == 0 || batch->total == 0 || NH == 0) return LTV_OK;
  LTV_REQUIRE(batch->total * NH < (int64_t(1) << 30), LTV_ERR_UNSUPPORTED,
              "too many new tokens in a call");
  const bool pages = batch->num_pages > 0;
  LTV_REQUIRE(q && out && q_strides && out_strides && k_page_strides && v_page_strides &&
                  (!pages || (k_pages && v_pages)),
              LTV_ERR_INVALID_ARG, "null pointer");
  const int es = elem_size(dtype), chunk = 16 / es;
  const AttnPlan p = plan_attention(*batch, NH, NKVH, max_len);
  LTV_REQUIRE(workspace_bytes >= part_bytes(p, D) && (p.nsplit <= 1 || workspace),
              LTV_ERR_WORKSPACE, "workspace too small");
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
             (uint32_t)(v_page_strides[2] / chunk), NH, NKVH, D, NH / NKVH, q_aligned ? 1 : 0,
             !rows_fit || batch->page_size % 16 != 0 ? 0 : batch->page_size % 64 == 0 ? 2 : 1, scale * kLog2e, p.tiles, p.group, p.chunk, p.nsplit, p.rows_cap,
             p.by_token, p.part_rows};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i] * es;
    a.os[i] = out_strides[i] * es;
  }
  const int64_t seqs = (int64_t)batch->B * NKVH;
  const int64_t units = seqs * p.nsplit * ((p.tiles + p.group - 1) / p.group);
  const int64_t grid = (units + 7) / 8 * 8 * p.group, joins = p.joins;
  LTV_REQUIRE(grid < (int64_t(1) << 31) && joins < (int64_t(1) << 30), LTV_ERR_UNSUPPORTED,
              "too many workgroups");
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kAttnThreads), 0, st, a);
  };
  auto by_width = [&](auto type) {
    using T = decltype(type);
    if (D == 64) launch(attn_tile_kernel<T, 64, false>);
    else if (D < 64) launch(attn_tile_kernel<T, 64, true>);
    else if (D == 128) launch(attn_tile_kernel<T, 128, false>);
    else launch(attn_tile_kernel<T, 128, true>);
  };
  if (dtype == LTV_DTYPE_F32) by_width(float()); else by_width(bf16_t());
  LTV_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    auto join = [&](auto type) {
      using T = decltype(type);
      if (p.nsplit <= 16)
        hipLaunchKernelGGL((attn_join_kernel<T, 1>), dim3((unsigned)((joins + 3) / 4)), dim3(256),
                           0, st, a);
      else if (p.nsplit <= 64)
        hipLaunchKernelGGL((attn_join_kernel<T, 4>), dim3((unsigned)joins), dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL((attn_join_kernel<T, 16>), dim3((unsigned)joins), dim3(1024), 0, st, a);
    };
    if (dtype == LTV_DTYPE_F32) join(float()); else join(bf16_t());
    LTV_LAUNCH_CHECK();
  }
  return LTV_OK;
}
