// Attention of new tokens over a paged cache held in 4 bits.
//
//   out[row] = sum_j p_j v_j,  p = softmax_{j <= pos(row)}(scale q[row] . k_j)
//
// k and v are the values that the codes and scales stand for, which bfloat16 holds exactly: the
// products are bfloat16 ones, and only queries and probabilities have parts (Split).
//
// Two kernels, by the rows that share a k/v head (few_rows).  Of few the reads are the bound, 17
// bytes for 32 channels: 16 sequences, one of 131,072 tokens, 6 k/v heads (500 MB) 96 us, 5.2 TB/s, the
// vector units issuing in half of the cycles.  Of many the products are, and the conversions and
// exponentials beside them: 8,193 tokens over 16,000 (0.51 TFLOP) 770 us, 657 TFLOP/s, the second
// parts of the probabilities, another 0.25, not counted; matrix units busy in 42 % of the cycles,
// vector units in 47 %, seldom both.  Scores, maxima, sums and outputs are float32.  The values are
// converted anew for each row tile; converted once, into a workspace of 16 bits that all of them
// read, is not built.
#include "../../include/nanochat_decoding_amd.h"
#include "ltv_fp4.hpp"
#include "ltv_paged_line.hpp"

namespace ltv {
namespace {

// Keys and values of 4-bit pages, for rows_one_by_one.
struct Fp4Pages {
  static __device__ __forceinline__ void load(const char* block, const AttnArgs& a, uint32_t in,
                                              int c, float (&x)[8], int shift) {
    const int size = a.batch.div.size;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(block + in * (a.D / 2) + c * 4);
    const float s = scale_bits((uint8_t)block[size * (a.D / 2) + (c >> 2) * size + in]);
    unpack16(fp4_eight(codes, s), x, bf16_t());
    if (shift != 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e], -shift);
  }
  static __device__ __forceinline__ void keys(const AttnArgs& a, int kvh, int page, uint32_t in,
                                              int c, float (&x)[8]) {
    load(a.k + kvh * a.kh + (uint64_t)((uint32_t)page * (uint64_t)a.kp) * 16, a, in, c, x, 0);
  }
  static __device__ __forceinline__ void values(const AttnArgs& a, int kvh, int page, uint32_t in,
                                                int c, float (&x)[8], int shift) {
    load(a.v + kvh * a.vh + (uint64_t)((uint32_t)page * (uint64_t)a.vp) * 16, a, in, c, x, shift);
  }
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// How many bfloat16 numbers stand for a query's element and for a probability.  Keys and values
// are such numbers themselves, so products are exact: a bfloat16 query is one, a float32 one the
// three of 8 bits each that its 24 are.  A probability rounded to one would be off by up to 2^-8, as
// much again as a bfloat16 output is by its own rounding; two leave 2^-16, three its float32 rounding.
template <typename T>
struct Split {
  static constexpr int kQuery = sizeof(T) == 2 ? 1 : 3, kProb = sizeof(T) == 2 ? 2 : 3;
};

// Eight float32 numbers' parts: bits of bfloat16, cut off and not rounded, so that no part passes
// the range and what is left is exact.
__device__ __forceinline__ void split_eight(const float (&x)[8], uint4 (&out)[3]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < 3; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = __float_as_uint(rest[2 * i]), hi = __float_as_uint(rest[2 * i + 1]);
      w[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
      rest[2 * i] -= __uint_as_float(lo & 0xffff0000u);
      rest[2 * i + 1] -= __uint_as_float(hi & 0xffff0000u);
    }
    out[n] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Eight probabilities' parts: bfloat16, two rounded ones; float32, three as above.
template <typename T>
__device__ __forceinline__ void split_probs(const float (&p)[8], uint4 (&out)[Split<T>::kProb]) {
  if constexpr (sizeof(T) == 4) {
    split_eight(p, out);
  } else {
    uint32_t w[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = cvt_pk_bf16(p[2 * i], p[2 * i + 1]);
      r[i] = cvt_pk_bf16(p[2 * i] - __uint_as_float(w[i] << 16),
                         p[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u));
    }
    out[0] = make_uint4(w[0], w[1], w[2], w[3]);
    out[1] = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// Eight elements of a query from element `at` on, in parts.
template <typename T>
__device__ __forceinline__ void load_query(const char* q, int at, uint4 (&out)[Split<T>::kQuery]) {
  if constexpr (sizeof(T) == 2) {
    __builtin_memcpy(&out[0], reinterpret_cast<const T*>(q) + at, 16);
  } else {
    float x[8];
    __builtin_memcpy(x, reinterpret_cast<const T*>(q) + at, 32);
    split_eight(x, out);
  }
}

__device__ __forceinline__ f32x4 product16(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// (the four lanes 16 apart)
__device__ __forceinline__ float across_quarters_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return across_halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// Bits of those of four scale bytes that are 192 or more: of values from 2^64 on, whose sums over
// many keys might pass the range, or of a NaN.  Rows of tiles with such are computed again one by
// one, with sums that are held 2^-60 smaller and each key left alone by rows that do not see it.
__device__ __forceinline__ uint32_t large_scales(uint32_t w) { return w & (w << 1) & 0x80808080u; }
constexpr int kShift = 60;

// ---------------------------------------------------------------------------
// Few rows: 16 of a row tile
// ---------------------------------------------------------------------------
// Each wavefront takes 32 keys of a block of 128 by itself, from memory into registers, and keeps
// its own maxima, sums and outputs; they are joined through LDS at the end of a piece.
//
// A wavefront has one tile of keys in registers, refilled as it is used: with three workgroups
// to a unit the others' reads are under way meanwhile.  (16 sequences as above, a call: 270 us
// with a second set of registers, which spills, 108 so.  Two or three tiles ahead in LDS 113,
// and 64 keys a step 125, for the registers and barriers they take; the rests of probabilities
// only where one weighs much, a branch that spills, 123.  The same reads without any conversions
// or products took 104 where all of it took 113.)  Beside the bytes a call pays for its start,
// the joining of wavefronts and the second kernel: 96 sequences of up to 6,000 tokens, 4 k/v
// heads of 64 with 8 rows each (62 MB), 27 + 6 us, four of up to 600 tokens 8 + 4.
//
// Products of 16 x 16 blocks.  S^T = K Q^T: a lane has 8 channels of a key in each step, and the
// order of the channels is free as long as the queries have it too: a lane takes D / 4 channels
// that follow each other, one load.  O^T = V^T P^T: the order of the keys is that in which the
// scores come, and the lane's channels of V are D / 16 that follow each other: one load for each
// of eight keys, whose values are put beside each other in pairs.
template <typename T, int D>
struct FewTile {
  static constexpr int kSteps = D / 32;                 // of the scores' products
  static constexpr int kScales = D == 96 ? 3 : 1;       // of a lane's channels of a key
  static constexpr int kLanes = D == 96 ? 12 : 16;      // with channels of V
  static constexpr int kCh = D / kLanes;                // of a lane
  uint32_t k[2][kSteps], ks[2][kScales];
  uint32_t v[8], vs[2];
};

constexpr int kFewRows = 16, kFewKeys = 128, kFewThreads = 256;
// Workgroups of a compute unit, as their registers allow.  (bfloat16, 64 sequences of 8,000 tokens
// and 4 heads of 128: two 54 us, three 51, four, which spill, 61; 16 heads of 32: three 105, four 98.
// float32, 8 heads of 64: two 77, three 66.)
constexpr int few_each(bool f32, int D) { return f32 ? (D <= 64 ? 3 : 2) : D <= 32 ? 4 : 3; }
template <typename T, int D>
constexpr int kFewEach = few_each(sizeof(T) == 4, D);

template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads, (kFewEach<T, D>))
    attn4_few_kernel(const AttnArgs a) {
  using Tile = FewTile<T, D>;
  constexpr int kSteps = Tile::kSteps, kCh = Tile::kCh, kQ = Split<T>::kQuery,
                kP = Split<T>::kProb;
  constexpr int kPitch = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[4 * kFewRows * kPitch];
  __shared__ float2 lds_ml[4 * kFewRows];
  static_assert(sizeof(lds_o) >= 16 * 130 * sizeof(float), "room for rows_one_by_one");

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto piece = [&](const PagedSeq& s, int b, int kvh, int tile, int begin, int end,
                   int64_t part0) {
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const char* kbase = a.k + (int64_t)kvh * a.kh;
    const char* vbase = a.v + (int64_t)kvh * a.vh;
    const int size = a.batch.div.size, vc = min(c, Tile::kLanes - 1) * kCh;
    const int row0 = tile * kFewRows, rows = min(s.n * a.g - row0, kFewRows);
    const bool row_ok = c < rows;
    const int t = row_ok ? a.by_g.quot(row0 + c) : 0;
    const int h = kvh * a.g + (row_ok ? row0 + c - t * a.g : 0);
    const int pos = row_ok ? s.len - s.n + t : -1;
    const int first_pos = s.len - s.n + a.by_g.quot(row0);  // of the tile's rows

    // (offsets of the lane from what is the same for all: bases in scalar registers)
    const uint32_t koff = c * (D / 2) + j * (D / 8), voff = 4 * j * (D / 2) + vc / 2;
    const uint32_t vsoff = vc / 32 * size + 4 * j;
    uint32_t ksoff[Tile::kScales];
#pragma unroll
    for (int e = 0; e < Tile::kScales; ++e) ksoff[e] = (j * (D / 4) + 8 * e) / 32 * size + c;
    // The pages of the 32 keys from kt on, looked up a tile ahead of their use.
    auto look_up = [&](int kt, int (&page)[2]) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
        page[half] = page_at(s.table, min(a.batch.div.quot(kt + 16 * half), a.batch.W - 1));
    };
    // Where the 16 keys from `at` on are, and how many there are.
    struct Place {
      const char *k, *v;  // their page's block
      uint32_t in;
      int n;
    };
    auto place = [&](int at, int page) {
      const bool ok = page >= 0 && page < a.batch.P && at < end;
      const uint32_t from = ok ? (uint32_t)page : 0u;
      return Place{kbase + (uint64_t)from * a.kp * 16, vbase + (uint64_t)from * a.vp * 16,
                   ok ? (uint32_t)(at - a.batch.div.quot(at) * size) : 0u, ok ? min(16, end - at) : 0};
    };
    Tile x;
    auto load_keys = [&](const Place (&p)[2]) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* codes = p[half].k + p[half].in * (D / 2);
        const char* scales = p[half].k + size * (D / 2) + p[half].in;
        __builtin_memcpy(x.k[half], reinterpret_cast<const uint32_t*>(codes + koff), D / 8);
#pragma unroll
        for (int e = 0; e < Tile::kScales; ++e) x.ks[half][e] = (uint8_t)scales[ksoff[e]];
      }
    };
    auto load_values = [&](const Place (&p)[2]) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* codes = p[half].v + p[half].in * (D / 2);
        const char* scales = p[half].v + size * (D / 2) + p[half].in;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const char* from = codes + voff + e * (D / 2);
          if constexpr (kCh == 8) x.v[4 * half + e] = *reinterpret_cast<const uint32_t*>(from);
          if constexpr (kCh == 4) x.v[4 * half + e] = *reinterpret_cast<const uint16_t*>(from);
          if constexpr (kCh == 2) x.v[4 * half + e] = *reinterpret_cast<const uint8_t*>(from);
        }
        x.vs[half] = *reinterpret_cast<const uint32_t*>(scales + vsoff);
      }
    };

    int pages[2] = {0, 0}, n[2] = {0, 0};
    int kt = begin + 32 * wave;
    if (kt < end) {
      look_up(kt, pages);
      const Place at[2] = {place(kt, pages[0]), place(kt + 16, pages[1])};
      load_keys(at);
      load_values(at);
      n[0] = at[0].n;
      n[1] = at[1].n;
      look_up(kt + kFewKeys, pages);
    }

    uint4 q[kSteps][kQ];
    {
      const int64_t trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;
      const char* from = a.q + (a.batch.starts != nullptr ? trow * a.qs[1]
                                                          : b * a.qs[0] + t * a.qs[1]) + h * a.qs[2];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
#pragma unroll
        for (int n = 0; n < kQ; ++n) q[i][n] = make_uint4(0, 0, 0, 0);
        if (row_ok) load_query<T>(from, j * (D / 4) + 8 * i, q[i]);
      }
    }

    f32x4 o[kCh];
#pragma unroll
    for (int d = 0; d < kCh; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys
    int again = 0;
    uint32_t large = 0;
    // The next tile's keys and values take the place of this one's as soon as those are used.
    for (; kt < end; kt += kFewKeys) {
      f32x4 sc[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sc[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint4 k = fp4_eight(x.k[half][i], scale_bits(x.ks[half][Tile::kScales == 1 ? 0 : i]));
#pragma unroll
          for (int n = 0; n < kQ; ++n) sc[half] = product16(k, q[i][n], sc[half]);
        }
      }
      in_order();
      const Place next[2] = {place(kt + kFewKeys, pages[0]), place(kt + kFewKeys + 16, pages[1])};
      const bool more = kt + kFewKeys < end;
      if (more) load_keys(next);
      // (a full tile that every row sees needs none of this)
      if (n[0] + n[1] < 32 || kt + 31 > first_pos) {
        // (keys that are not there have no values: whatever their bytes are must not come in as 0
        // times NaN)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t there = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 4 * j + i;
            if (key < n[half]) there |= 255u << (8 * i);
            if (key >= n[half] || kt + 16 * half + key > pos) sc[half][i] = -INFINITY;
          }
          x.vs[half] &= there;
        }
      }
      large |= large_scales(x.vs[0]) | large_scales(x.vs[1]);
      float top = sc[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[i / 4][i % 4]);
      top = across_quarters_max(top) * a.scale;
      // the maximum in use stays until a score passes it by a factor of 2^8
      if (__any(top > m + 8.0f)) {
        const float mn = fmaxf(m, top);
        // (from here on the argument of an exponential is off by 2^-6 and more)
        if (__any(fabsf(mn) > 0x1p18f && mn != -INFINITY)) again = 1;
        const float was = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= was;
#pragma unroll
        for (int d = 0; d < kCh; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] *= was;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i / 4][i % 4], a.scale, -base));
        l += p[i];
      }
      uint4 pw[kP];
      split_probs<T>(p, pw);
      // V: two channels of eight keys, and of each channel the keys beside each other
      float scale[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) scale[e] = scale_bits(x.vs[e / 4] >> (8 * (e % 4)) & 255u);
      auto channels = [&](auto of) {
        constexpr int kOf = decltype(of)::value;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = fp4_pair<kOf>(x.v[e], scale[e]);
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t sel = odd ? 0x07060302u : 0x05040100u;
          const uint4 v = make_uint4(
              __builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
              __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel));
#pragma unroll
          for (int n = 0; n < kP; ++n) o[2 * kOf + odd] = product16(v, pw[n], o[2 * kOf + odd]);
        }
      };
      channels(std::integral_constant<int, 0>());
      if constexpr (kCh >= 4) channels(std::integral_constant<int, 1>());
      if constexpr (kCh == 8) {
        channels(std::integral_constant<int, 2>());
        channels(std::integral_constant<int, 3>());
      }
      in_order();
      if (more) {
        load_values(next);
        n[0] = next[0].n;
        n[1] = next[1].n;
        look_up(kt + 2 * kFewKeys, pages);
      }
    }

    if (__syncthreads_or(again | (int)large)) {
      const int shift = __syncthreads_or((int)large) ? kShift : 0;
      rows_one_by_one<T, kFewThreads, Fp4Pages>(a, s, b, kvh, row0, row0 + rows, begin, end, part0,
                                                lds_o, shift);
      __syncthreads();
      return;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (j == 0) lds_ml[wave * kFewRows + c] = make_float2(m, l);
    barrier();
    {
      float mx = m;
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, lds_ml[w * kFewRows + c].x);
      const float f = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.0f : mx));
      // (column c of a block is a row, its rows 4 j .. groups of kCh channels)
      if (row_ok)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((4 * j + i) * kCh >= D) continue;
          float* to = lds_o + (wave * kFewRows + c) * kPitch + (4 * j + i) * kCh;
#pragma unroll
          for (int d = 0; d < kCh; ++d) to[d] = o[d][i] * f;
        }
    }
    barrier();
    for (int i = threadIdx.x; i < rows * (D / 4); i += kFewThreads) {
      const int r = i / (D / 4), ch = (i - r * (D / 4)) * 4;
      float mx = -INFINITY, sum = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, lds_ml[w * kFewRows + r].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 ml = lds_ml[w * kFewRows + r];
        sum = fmaf(ml.y, __builtin_amdgcn_exp2f(ml.x - (mx == -INFINITY ? 0.0f : mx)), sum);
        const float4 x = *reinterpret_cast<const float4*>(lds_o + (w * kFewRows + r) * kPitch + ch);
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      const int tt = a.by_g.quot(row0 + r), hh = kvh * a.g + row0 + r - tt * a.g;
      if (part0 >= 0) {
        *reinterpret_cast<float4*>(a.part + (part0 + r) * D + ch) = acc;
        if (ch == 0) part_ml(a)[part0 + r] = make_float2(mx, sum);
      } else {
        const int64_t trow = a.batch.starts != nullptr ? s.row0 + tt : (int64_t)b * a.batch.T + tt;
        char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                       : b * a.os[0] + tt * a.os[1]) + hh * a.os[2];
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2*>(out + ch * 2) =
              make_uint2(cvt_pk_bf16(acc.x * inv, acc.y * inv), cvt_pk_bf16(acc.z * inv, acc.w * inv));
        else
          *reinterpret_cast<float4*>(out + ch * 4) =
              make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (ch == 0 && a.lse != nullptr)
          a.lse[trow * a.NH + hh] =
              sum == 0.0f ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * kLn2;
      }
    }
    barrier();  // (LDS is read)
  };
  walk_line<kFewKeys, false, kFewThreads, kFewRows, 256 * kFewEach<T, D>, const AttnArgs&>(a, piece);
}

// ---------------------------------------------------------------------------
// Many rows: 128 of a row tile
// ---------------------------------------------------------------------------
// 32 rows to each of four wavefronts, and tiles of 64 keys that they share: each thread turns a
// sixteenth of a token's channels of K and of V into bfloat16 and puts them into LDS, a tile ahead
// of the products.  Those are in 32 x 32 blocks, S^T = K Q^T and O^T = V^T P^T as over 16-bit
// pages: a lane holds 16 keys of one row, and its probabilities are, without any exchange, the
// right-hand operand of the second product (ds_read_b64_tr_b16 transposes four keys of a column).
// float32 has three products for each (of the queries' parts and of the probabilities'), and one
// workgroup to a unit for the registers: a prompt of 4,096 tokens 116 us with the joining, 222 TFLOP/s
// counted once, where a float32 product of two large matrices reaches 154.
constexpr int kManyRows = 128, kManyKeys = 64, kManyThreads = 256;
template <typename T>
constexpr int kManyEach = sizeof(T) == 2 ? 2 : 1;  // workgroups of a compute unit

// Rows of DP channels (D padded with zeros) in LDS; chunk c (8 channels) of row r sits in a slot
// chosen so that the lanes of one read fall on different banks: of K 16 consecutive rows, one
// chunk each, of V four rows, 64 bytes each.
template <int DP>
struct ManyTile {
  static constexpr int kChunks = DP / 8, kPhase = kChunks < 16 ? 2 : 1;
  static constexpr int kUnits = kManyKeys * kChunks, kRow = kChunks * 16, kBytes = kUnits * 16;
  static __device__ __forceinline__ int k_slot(int r, int c) {
    return r * kChunks + (c ^ ((r / kPhase) & (kChunks - 1)));
  }
  static __device__ __forceinline__ int v_swizzle(int r) {
    return ((r / kPhase) & (4 / kPhase - 1)) * 4;
  }
  static __device__ __forceinline__ int v_slot(int r, int c) {
    return r * kChunks + (c ^ v_swizzle(r));
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 product32(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T, int D>
__global__ void __launch_bounds__(kManyThreads, kManyEach<T>) attn4_many_kernel(const AttnArgs a) {
  constexpr int DP = D <= 64 ? 64 : 128;
  using Ti = ManyTile<DP>;
  constexpr int KT = kManyKeys, KB = KT / 32, kSteps = DP / 16, kDB = DP / 32;
  constexpr int kQ = Split<T>::kQuery, kP = Split<T>::kProb;
  constexpr int NC = D / 32, NS = D == 96 ? 3 : 1;  // chunks and scales of a thread's channels
  __shared__ uint4 lds[4 * Ti::kUnits];             // K, V, and again
  static_assert(sizeof(lds) >= 16 * 130 * sizeof(float), "room for rows_one_by_one");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  auto zero_padding = [&]() {
    if constexpr (D != DP) {
      constexpr int kPad = Ti::kChunks - D / 8;
      for (int i = threadIdx.x; i < 2 * KT * kPad; i += kManyThreads) {
        const int buf = i / (KT * kPad), r = i / kPad % KT, c = D / 8 + i % kPad;
        lds[buf * 2 * Ti::kUnits + Ti::k_slot(r, c)] = make_uint4(0, 0, 0, 0);
        lds[(buf * 2 + 1) * Ti::kUnits + Ti::v_slot(r, c)] = make_uint4(0, 0, 0, 0);
      }
    }
  };
  zero_padding();

  auto piece = [&](const PagedSeq& s, int b, int kvh, int tile, int begin, int end,
                   int64_t part0) {
    const char* kbase = a.k + (int64_t)kvh * a.kh;
    const char* vbase = a.v + (int64_t)kvh * a.vh;
    const int size = a.batch.div.size;
    // (opaque: what follows from the lane is not kept in registers around the pieces)
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, ln = lane & 31, hf = lane >> 5;
    // The page of the lane-th key of a tile, -1: none or past the end.
    auto page_of = [&](int kt) {
      const int at = kt + lane;
      const int page = s.table[min(a.batch.div.quot(at), a.batch.W - 1)];
      return at < end && page < a.batch.P ? page : -1;
    };
    // A thread's part of a tile: a quarter of the channels of key thread / 4.
    const int key = thread >> 2, quarter = thread & 3;
    // The chunks in an order that has the writes of eight lanes (two keys) on different banks, which
    // the swizzles that the reads need do not.  (In order the conflicts cost 14 % of the cycles of a
    // long prompt.)
    const int kturn = NC == 4 ? quarter & 2 : NC == 2 ? key & 1 : 0;
    const int vturn = NC == 4 ? (quarter & 2) | (key & 1) : kturn;
    uint32_t kc[NC], vc[NC], ks[NS], vs[NS];
    auto load = [&](int kt, int pages) {
      const int page = __shfl(pages, key), at = kt + key;
      const bool ok = page >= 0;
      const uint32_t in = ok ? (uint32_t)(at - a.batch.div.quot(at) * size) : 0u;
      const uint32_t from = ok ? (uint32_t)page : 0u;
      const char* kb = kbase + (uint64_t)(from * a.kp) * 16;
      const char* vb = vbase + (uint64_t)(from * a.vp) * 16;
      const uint32_t codes = in * (D / 2) + quarter * (D / 8);
#pragma unroll
      for (int e = 0; e < NC; ++e) {
        kc[e] = *reinterpret_cast<const uint32_t*>(kb + codes + (e ^ kturn) * 4);
        vc[e] = *reinterpret_cast<const uint32_t*>(vb + codes + (e ^ vturn) * 4);
      }
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        const uint32_t scale = size * (D / 2) + (quarter * NC + e) / 4 * size + in;
        ks[e] = (uint8_t)kb[scale];
        vs[e] = (uint8_t)vb[scale];
      }
    };
    uint32_t large = 0;
    // Part x of a tile into LDS: chunk x / 2 of K or V.  (A key that is not there is 0: whatever its
    // bytes are must not come in as 0 times NaN.)
    constexpr int kParts = 2 * NC;
    auto store = [&](int x, bool ok, int buf) {
      const int e = x / 2, n = NS == 1 ? 0 : e, c = quarter * NC;
      uint4* to = lds + buf * 2 * Ti::kUnits;
      if (x % 2 == 0) {
        to[Ti::k_slot(key, c + (e ^ kturn))] =
            fp4_eight(ok ? kc[e] : 0u, ok ? scale_bits(ks[n]) : 1.0f);
      } else {
        if (e < NS) large |= ok ? large_scales(vs[e]) : 0u;
        to[Ti::kUnits + Ti::v_slot(key, c + (e ^ vturn))] =
            fp4_eight(ok ? vc[e] : 0u, ok ? scale_bits(vs[n]) : 1.0f);
      }
    };

    // the first tile into LDS, the second on its way, the pages of the third
    uint64_t there = 0, next = 0;
    int page = -1;
    if (begin < end) {
      page = page_of(begin);
      load(begin, page);
      next = __ballot(page >= 0);
      page = page_of(begin + KT);
    }

    // (Of few rows one wavefront has all products: not on the same SIMD in both workgroups.)
    const int wrow = tile * kManyRows +
                     ((wave + (int)(blockIdx.x / (128 * kManyEach<T>)) * 2) & 3) * 32;
    const int rows = s.n * a.g, row = wrow + ln;
    const bool row_ok = row < rows;
    const int t = row_ok ? a.by_g.quot(row) : 0;
    const int h = kvh * a.g + (row_ok ? row - t * a.g : 0);
    const int pos = row_ok ? s.len - s.n + t : -1;
    const int64_t trow = a.batch.starts != nullptr ? s.row0 + t : (int64_t)b * a.batch.T + t;
    // the last position that any row of the wavefront sees, and the first one's
    const bool wave_on = wrow < rows;
    const int wave_end = wave_on ? s.len - s.n + a.by_g.quot(min(wrow + 31, rows - 1)) + 1 : 0;
    const int wave_min = wave_on ? s.len - s.n + a.by_g.quot(wrow) : 0;

    uint4 q[kQ][kSteps];
    {
      const char* from = a.q + (a.batch.starts != nullptr ? trow * a.qs[1]
                                                          : b * a.qs[0] + t * a.qs[1]) + h * a.qs[2];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        uint4 parts[kQ];
#pragma unroll
        for (int n = 0; n < kQ; ++n) parts[n] = make_uint4(0, 0, 0, 0);
        if (row_ok && (2 * i + hf) * 8 < D) load_query<T>(from, (2 * i + hf) * 8, parts);
#pragma unroll
        for (int n = 0; n < kQ; ++n) q[n][i] = parts[n];
      }
    }

    // Where the lane reads K's row ln, and V's four rows from 4 hf, in the first buffer.  The
    // swizzles exclusive-or a slot, so a later step's chunk is an exclusive or away; rows further
    // on a constant.
    const uint32_t lds0 = lds_address(lds);
    const uint32_t kat = lds0 + Ti::k_slot(ln, hf) * 16;
    const int vr = 4 * hf + (lane & 15) / 4;
    const uint32_t vat = lds0 + Ti::kBytes +
                         Ti::v_slot(vr, ((lane >> 4) & 1) * 2 + (lane & 3) / 2) * 16 + (lane & 1) * 8;

    f32x16 o[kDB];
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys
    int again = 0;

    if (begin < end) {
      barrier();  // (the piece before is read to its end)
#pragma unroll
      for (int x = 0; x < kParts; ++x) store(x, next >> key & 1, 0);
      if (begin + KT < end) load(begin + KT, page);
    }
    int buf = 0;
    for (int kt = begin; kt < end; kt += KT, buf ^= 1) {
      there = next;
      barrier();  // this tile is there, and the other buffer is read
      // The next tile is put into LDS between the first products (all at once before them, its
      // conversions and writes cost a long prompt 28 % of its time), the one after it loaded then.
      const bool more = kt + KT < end, after = kt + 2 * KT < end;
      if (more) {
        next = __ballot(page >= 0);
        page = page_of(kt + 2 * KT);
      }
      const bool ok = next >> key & 1;
      if (kt >= wave_end) {
        if (more)
#pragma unroll
          for (int x = 0; x < kParts; ++x) store(x, ok, buf ^ 1);
        if (after) load(kt + 2 * KT, page);
        continue;
      }
      const uint32_t ka = kat + buf * 2 * Ti::kBytes, va = vat + buf * 2 * Ti::kBytes;
      f32x16 sc[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
      auto scores = [&](auto with_store) {
        constexpr int N = kSteps * KB, AHEAD = 5;
        uint4 kf[AHEAD];
        auto keys = [&](int n) {
          return __builtin_bit_cast(
              uint4, lds_read<u32x4>((ka ^ (32 * (n / KB))) + n % KB * 32 * Ti::kRow));
        };
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) kf[n] = keys(n);
        in_order();
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int e = 0; e < kQ; ++e) sc[n % KB] = product32(kf[n % AHEAD], q[e][n / KB], sc[n % KB]);
          if (n + AHEAD < N) kf[n % AHEAD] = keys(n + AHEAD);
          if constexpr (decltype(with_store)::value)
#pragma unroll
            for (int x = n * kParts / N; x < (n + 1) * kParts / N; ++x) store(x, ok, buf ^ 1);
          in_order();
        }
      };
      if (more) scores(std::true_type()); else scores(std::false_type());
      if (after) load(kt + 2 * KT, page);
      // keys that the lane's row sees, as bits from the lane half's first
      if (there != ~0ull || kt + KT - 1 > wave_min) {
        const int n = pos - kt + 1;  // keys up to the row's own
        const uint64_t seen = n <= 0 ? 0 : there & (n >= 64 ? ~0ull : (1ull << n) - 1);
        const uint64_t mine = seen >> (4 * hf);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((mine >> (kb * 32 + 8 * (i / 4) + i % 4)) & 1)) sc[kb][i] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[kb][i]);
      top = across_halves_max(top) * a.scale;
      // the maximum in use stays until a score passes it by a factor of 2^8
      if (__any(top > m + 8.0f)) {
        const float mn = fmaxf(m, top);
        // (from here on the argument of an exponential is off by 2^-6 and more)
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
      constexpr int N = KB * 2;  // steps of 16 keys
      uint4 vf[2][kDB];
      auto values = [&](int e, int d) {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        union {
          s16x4 half[2];
          uint4 v;
        } f;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          f.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4*)(uintptr_t)((va ^ (64 * d)) + (16 * e + 8 * x) * Ti::kRow));
        return f.v;
      };
      // Probabilities 2 x, 2 x + 1 of step e
      auto pair = [&](int e, int x) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int i = 8 * (e % 2) + 2 * x + y;
          const float v = __builtin_amdgcn_exp2f(fmaf(sc[e / 2][i], a.scale, -base));
          sc[e / 2][i] = v;
          l += v;
        }
      };
      // .. their first part in bfloat16, and what comes after part w (float32: in their place)
      auto first_part = [&](int e, int x) {
        const int i = 8 * (e % 2) + 2 * x;
        if constexpr (sizeof(T) == 2) return cvt_pk_bf16(sc[e / 2][i], sc[e / 2][i + 1]);
        return __builtin_amdgcn_perm(__float_as_uint(sc[e / 2][i + 1]),
                                     __float_as_uint(sc[e / 2][i]), 0x07060302);
      };
      auto part_after = [&](int e, int x, uint32_t w) {
        const int i = 8 * (e % 2) + 2 * x;
        const float p0 = sc[e / 2][i] - __uint_as_float(w << 16);
        const float p1 = sc[e / 2][i + 1] - __uint_as_float(w & 0xffff0000u);
        if constexpr (sizeof(T) == 2) return cvt_pk_bf16(p0, p1);
        sc[e / 2][i] = p0;
        sc[e / 2][i + 1] = p1;
        return __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302);
      };
      // Step e: the products of the first parts, then those of the rests, the next step's
      // probabilities between them.  (bfloat16 without the rests, 8,193 tokens over 16,000: 745 us
      // for 800 a call.)
      uint32_t w[kP][4], ahead[kP][4];
      auto split = [&](int e, int x, uint32_t (&to)[kP][4]) {
        pair(e, x);
        to[0][x] = first_part(e, x);
#pragma unroll
        for (int n = 1; n < kP; ++n) to[n][x] = part_after(e, x, to[n - 1][x]);
      };
#pragma unroll
      for (int d = 0; d < kDB; ++d) vf[0][d] = values(0, d);
#pragma unroll
      for (int x = 0; x < 4; ++x) split(0, x, w);
      in_order();
#pragma unroll
      for (int e = 0; e < N; ++e) {
#pragma unroll
        for (int n = 0; n < kP; ++n)
#pragma unroll
          for (int d = 0; d < kDB; ++d) {
            o[d] = product32(vf[e & 1][d], make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]), o[d]);
            if (e + 1 < N) {
              const int at = n * kDB + d;
              if (n == 0) vf[(e + 1) & 1][d] = values(e + 1, d);
#pragma unroll
              for (int x = at * 4 / (kDB * kP); x < (at + 1) * 4 / (kDB * kP); ++x)
                split(e + 1, x, ahead);
            }
            in_order();
          }
#pragma unroll
        for (int n = 0; n < kP; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) w[n][x] = ahead[n][x];
      }
    }

    if (__syncthreads_or(again | (int)large)) {
      const int shift = __syncthreads_or((int)large) ? kShift : 0;
      rows_one_by_one<T, kManyThreads, Fp4Pages>(a, s, b, kvh, tile * kManyRows,
                                                 min(rows, (tile + 1) * kManyRows), begin, end,
                                                 part0, reinterpret_cast<float*>(lds), shift);
      __syncthreads();
      zero_padding();
      return;
    }
    l += __shfl_xor(l, 32);
    if (!row_ok) return;
    if (part0 >= 0) {
      const int64_t at = part0 + row - tile * kManyRows;
      float* po = a.part + at * D;
#pragma unroll
      for (int d = 0; d < kDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int ch = d * 32 + 2 * i + 4 * hf;
          if (ch < D)
            *reinterpret_cast<float4*>(po + ch) =
                make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
        }
      if (hf == 0) part_ml(a)[at] = make_float2(m, l);
      return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    char* out = a.out + (a.batch.starts != nullptr ? trow * a.os[1]
                                                   : b * a.os[0] + t * a.os[1]) + h * a.os[2];
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int ch = d * 32 + 2 * i + 4 * hf;
        if (ch >= D) continue;
        const float x[4] = {o[d][i] * inv, o[d][i + 1] * inv, o[d][i + 2] * inv, o[d][i + 3] * inv};
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2*>(out + ch * 2) =
              make_uint2(cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]));
        else
          *reinterpret_cast<float4*>(out + ch * 4) = make_float4(x[0], x[1], x[2], x[3]);
      }
    if (hf == 0 && a.lse != nullptr)
      a.lse[trow * a.NH + h] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  };
  walk_line<KT, false, kManyThreads, kManyRows, 256 * kManyEach<T>, const AttnArgs&>(a, piece);
}

// Up to how many rows of a k/v head tiles of 16 read every key for themselves: 16 sequences of
// 4,000 tokens, 4 heads with 32 rows 39 us in tiles of 16 and 45 in one of 128, with 64 rows 48 and
// 54, with 128 rows 70 and 64.
constexpr int kMostFewRows = 64;

// Of more rows, calls so small that tiles of 128 would be cut into pieces of a few keys, for the
// whole card to have some: by rows of all heads times the longest sequence, and in float32, whose
// tiles of 128 have one workgroup to a unit, also by rows alone.  (In tiles of 128 and of 16 us,
// 6 heads of 128: bfloat16, 512 tokens over 2,000 41 and 34, 2,048 alone 47 and 42, 1,024 over 8,000
// 75 and 87, 16 chunks of 128 over up to 2,000 with 8 heads of 64 42 and 44; float32, 512 over 2,000 44
// and 37, five chunks of up to 600 over up to 4,000 among three single tokens 67 and 61, 1,024 over
// 8,000 110 and 113, 2,048 alone 58 and 68.)
bool few_rows(bool f32, int64_t rows, double all_rows, double max_len) {
  return rows <= kMostFewRows || all_rows * max_len <= (f32 ? 0x1p24 : 0x1p25) ||
         (f32 && all_rows <= 8192);
}

AttnPlan plan_attention4(const ltv_paged_batch& b, int dtype, int NH, int NKVH, int D,
                         int max_len) {
  const bool f32 = dtype == LTV_DTYPE_F32;
  const int64_t rows = (int64_t)std::max(b.T, 1) * (NH / NKVH);
  LineShape shape{};
  const bool few = few_rows(f32, rows, (double)b.total * NH, max_len);
  if (few) {
    shape.keys = kFewKeys;
    shape.log_rows = 4;
    shape.grid = 256 * few_each(f32, D);
    shape.group = 1;
    shape.least = 1;
  } else {
    const int64_t tiles = (rows + kManyRows - 1) / kManyRows;
    shape.keys = kManyKeys;
    shape.log_rows = 7;
    shape.grid = 256 * (f32 ? kManyEach<float> : kManyEach<bf16_t>);
    shape.group = f32 ? 1 : tiles >= 3 ? 4 : (int)tiles;
    shape.least = 2;
  }
  AttnPlan p = plan_line(b, NH, NKVH, D, max_len, shape);
  p.few = few;
  // (row tiles of 16 count alike on the line, as those in the middle of the longest chunk)
  if (few) p.group_tokens = std::max(p.group_tokens, b.T / 2);
  return p;
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_paged_attention_fp4_workspace_size(int dtype, const ltv_paged_batch* batch,
                                                         int NH, int NKVH, int D, int max_len) {
  if (batch == nullptr || batch->B <= 0 || batch->T < 0 || NKVH <= 0 || NH < NKVH || D <= 0)
    return 0;
  return plan_attention4(*batch, dtype, NH, NKVH, D, max_len).bytes;
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
  bool out_ok = aligned16(out);
  for (int i = batch->starts != nullptr ? 1 : 0; i < 3; ++i)
    out_ok = out_ok && out_strides[i] * es % 16 == 0;
  LTV_REQUIRE(out_ok, LTV_ERR_UNSUPPORTED, "the output's rows must be 16-byte aligned");
  const AttnPlan p = plan_attention4(*batch, dtype, NH, NKVH, D, max_len);
  LTV_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= p.bytes, LTV_ERR_WORKSPACE,
              "workspace too small");
  AttnArgs a{PagedBatch(*batch), (const char*)q, (const char*)k_pages, (const char*)v_pages,
             (char*)out, lse, (float*)workspace, {}, {},
             pages ? k_page_strides[1] : 0, pages ? v_page_strides[1] : 0,
             pages ? (uint32_t)(k_page_strides[0] / 16) : 0, 0,
             pages ? (uint32_t)(v_page_strides[0] / 16) : 0, 0, NH, NKVH, D, NH / NKVH, 0,
             1, 0, scale * kLog2e, p.group == 4 ? 2 : p.group - 1, p.ranges,
             p.least, p.unit, p.group_tokens, p.slope, p.extra, p.log_rows, p.part_tile,
             PageDiv(NH / NKVH), PageDiv(p.ranges), p.part_rows, nullptr, nullptr};
  a.cuts = (Cut*)((char*)workspace + p.cuts_at);
  a.head = (int*)(a.cuts + (size_t)p.ranges * p.group);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i] * es;
    a.os[i] = out_strides[i] * es;
  }
  const unsigned grid = p.ranges * p.group;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto type, auto width) {
    using T = decltype(type);
    constexpr int W = decltype(width)::value;
    if (p.few)
      hipLaunchKernelGGL((attn4_few_kernel<T, W>), dim3(grid), dim3(kFewThreads), 0, st, a);
    else
      hipLaunchKernelGGL((attn4_many_kernel<T, W>), dim3(grid), dim3(kManyThreads), 0, st, a);
  };
  auto by_width = [&](auto type) {
    if (D == 32) launch(type, std::integral_constant<int, 32>());
    else if (D == 64) launch(type, std::integral_constant<int, 64>());
    else if (D == 96) launch(type, std::integral_constant<int, 96>());
    else launch(type, std::integral_constant<int, 128>());
  };
  if (dtype == LTV_DTYPE_F32) by_width(float()); else by_width(bf16_t());
  LTV_LAUNCH_CHECK();
  if (p.joins) {
    auto join = [&](auto type) {
      const int each = p.part_tile <= 16 ? 1 : 8;
      hipLaunchKernelGGL(attn_join_kernel<decltype(type)>,
                         dim3(grid, (p.part_tile + each - 1) / each), dim3(256), 0, st, a, each);
    };
    if (dtype == LTV_DTYPE_F32) join(float()); else join(bf16_t());
    LTV_LAUNCH_CHECK();
  }
  return LTV_OK;
}
