// Log probabilities of given tokens, entropy and top alternatives of rows of logits,
// and their gradient.
//
//   z = c tanh(x / c)  (or x),  m = max z,  S = sum e^{z - m},  A = sum (z - m) e^{z - m}
//   lse = m + log S,   logprob = z_t - lse,   entropy = log S - A / S
//
// With a cap up to 64, tanh(y) = 1 - 2 r with r = 1 / (1 + e^{2 y}): z = c - 2 c r lies in
// [-c, c], where e^z and the sum of 2^31 of them neither overflow nor vanish in float32, so 0
// serves as the maximum; z's derivative is 4 r (1 - r).  Its error is some roundings of c (of
// 15: 2e-6 at most), not of z, for half the instructions of a tanh.  With a larger cap z is
// c tanh(x / c) to its own last bits, and m is the row's maximum: 4,096 rows of 65,536
// bfloat16 logits with five alternatives take 224 us with a cap of 100 and 120 with one of
// 50, 4,096 of 50,257 with their gradient 388 and 256.
//
// Forward.  One pass over the logits: each thread keeps m, S and A of its elements and they
// are joined at the end.  A workgroup takes a row, or, where there are few rows, a piece of
// one; a second kernel then joins the pieces.  The alternatives are found in the same pass.
// The first elements (the lowest indices) are kept in registers; of the largest of each
// of 64 groups of them the k-th is a bound that at least k elements reach, so from there
// on only larger elements can be among the top k (an equal one has a higher index), a few
// k of them on usual rows.  They are collected and ranked at the end.  A row that has too
// many (a large vocabulary and k) is read again with the k-th of those collected as the bound.
// If they are too many still (the row rises along its indices) the bound is found digit by
// digit of the keys, counted in a reading each: eight at most, two or three as a rule, and one
// that collects.  512 such rows of 131,072 float32 take 477 us, shuffled ones 74.  Bounded by
// the reads: 4,096 rows of 65,536 bfloat16 logits with five alternatives 116 us, 4.6 TB/s; 16
// rows of float32 in 256 pieces 7 us, half of it latency.  (Keys of value and index for each of
// the first elements, not for the largest of a thread alone: 6 us more.)
//
// Backward.  Elementwise given lse; a workgroup takes a piece of a row and sets the
// elements of the target and the alternatives again, with their own terms.  4,096 rows of
// 50,257 bfloat16 logits about 150 us, 5.5 TB/s read and written.
#include <algorithm>
#include <type_traits>

#include "ltv_logprobs.hpp"

namespace ltv {
namespace {

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
  int piece, pieces;         // elements of a workgroup, workgroups of a row
  bool parts;                // a kernel joins the pieces: pieces > 1, or another's
  const uint8_t* skip;       // rows to leave out, or null
  float* part_sums;          // (N, pieces, 3), parts
  uint64_t* part_keys;       // (N, pieces, top_k)
};

// (below 2^-13 of the cap x (1 - (x / c)^2 / 3 + ..) rounds to x)
__device__ __forceinline__ float wide_capped(float x, float cap) {
  return fabsf(x) <= cap * 0x1p-13f ? x : cap * tanhf(x / cap);
}

template <Cap CAP>
__device__ __forceinline__ float capped(float x, float cap) {
  if constexpr (CAP == kNoCap) return x;
  if constexpr (CAP == kWideCap) return wide_capped(x, cap);
  return fmaf(-2.0f * cap, cap_r(x, cap_scale_of(cap)), cap);
}

// 16 bytes at any alignment of the element.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// m, S and A of some elements: S = sum 2^d, A = sum d 2^d with d = (x - m) log2(e) (the
// difference first: the logits may be of any size).  By r there is no m: S = sum e^z, and A
// counts r instead of d.
template <Cap CAP>
struct Sums {
  float m = -INFINITY, s = 0.0f, a = 0.0f;

  // S and A from another maximum w above the old, or from far below it (w 2^w -> 0)
  static __device__ __forceinline__ float moved_a(float d, float s, float a, float w) {
    return w == 0.0f ? s * 0.0f : fmaf(d, s, a) * w;  // (a NaN stays)
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&logits)[N], float cap) {
    if constexpr (CAP == kCap) {
      const float cap_scale = cap_scale_of(cap);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float r = cap_r(logits[i], cap_scale);
        const float e = cap_exp(r, cap);
        s += e;
        a = fmaf(r, e, a);
      }
    } else {
      using Z = std::conditional_t<CAP == kCap64 || CAP == kTanh64, double, float>;
      Z z[N];
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (std::is_same_v<Z, double>) z[i] = capped64<CAP>(logits[i], cap);
        else z[i] = capped<CAP>(logits[i], cap);
        x[i] = (float)z[i];
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
      if (top > m) {
        if (m != -INFINITY) {
          const float d = (m - top) * kLog2e, was = __builtin_amdgcn_exp2f(d);
          a = moved_a(d, s, a, was);
          s *= was;
        }
        m = top;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (float)(z[i] - (Z)base) * kLog2e;
        const float e = __builtin_amdgcn_exp2f(d);
        s += e;
        a = fmaf(fmaxf(d, -1000.0f), e, a);  // (-inf adds nothing; NaN comes by e)
      }
    }
  }
  __device__ __forceinline__ void join(float m2, float s2, float a2) {
    if constexpr (CAP == kCap) {
      s += s2;
      a += a2;
    } else {
      const float mn = fmaxf(m, m2);
      if (mn == -INFINITY) {
        s += s2;  // 0, or a NaN
        return;
      }
      const float d1 = (m - mn) * kLog2e, d2 = (m2 - mn) * kLog2e;
      const float w1 = __builtin_amdgcn_exp2f(d1), w2 = __builtin_amdgcn_exp2f(d2);
      a = moved_a(d1, s, a, w1) + moved_a(d2, s2, a2, w2);
      s = s * w1 + s2 * w2;
      m = mn;
    }
  }
};

constexpr int kGroups = 64;    // of the first elements: as many as top_k may be
constexpr int kCands = 1024;   // collected elements

constexpr int kThreads = 256, kWaves = kThreads / 64;

// What a row's sums make: log(sum of exponentials) and entropy.
template <Cap CAP>
__device__ __forceinline__ void row_results(const Sums<CAP>& sums, float cap, float& lse,
                                            float& entropy) {
  const float log_s = __builtin_amdgcn_logf(sums.s), a = sums.a / sums.s;
  lse = fmaf(log_s, kLn2, CAP == kCap ? 0.0f : sums.m);
  // (by r: the mean of z is c - 2 c a)
  entropy = CAP == kCap ? fmaf(log_s, kLn2, cap * fmaf(2.0f, a, -1.0f)) : (log_s - a) * kLn2;
}

// The target's logit (one thread reads it ahead), and the row's results that are not
// alternatives.
struct Target {
  bool given = false;
  float x = 0.0f;
};
template <typename T>
__device__ __forceinline__ Target target_of(const LogpArgs& p, int64_t n, const T* row) {
  Target t;
  const int64_t id = p.targets[n];
  t.given = id >= 0 && id < p.V;
  if (t.given) t.x = io_traits<T>::load(row + id);
  return t;
}
template <Cap CAP>
__device__ __forceinline__ void store_row(const LogpArgs& p, int64_t n, const Target& t,
                                          float lse, float entropy) {
  p.logprobs[n] = t.given ? capped<CAP>(t.x, p.cap) - lse : 0.0f;
  if (p.entropy != nullptr) p.entropy[n] = entropy;
  if (p.lse != nullptr) p.lse[n] = lse;
}

template <typename T, Cap CAP, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_forward_kernel(const LogpArgs p) {
  constexpr int N = io_traits<T>::kVec;
  constexpr int kFirst = 8192 / (kThreads * N);  // vectors of a thread kept for the bound
  constexpr int kAhead = 4;                      // loads in flight
  __shared__ float lds_sums[kWaves][3];
  __shared__ unsigned long long groups[TOP ? kGroups : 1];
  __shared__ unsigned long long cands[TOP ? kCands : 1];
  __shared__ unsigned long long bound_lds;
  __shared__ int count, above_lds;
  const int64_t n = blockIdx.x;
  if (p.skip != nullptr && p.skip[n] != 0) return;
  const int begin = blockIdx.y * p.piece;
  const T* whole_row = reinterpret_cast<const T*>(p.x) + n * p.xs;
  const T* row = whole_row + begin;
  const int tid = threadIdx.x, lane = tid & 63, V = min(p.V - begin, p.piece);
  const int whole = V / N;  // vectors that the piece fills; the rest are single elements
  Sums<CAP> sums;
  float bound = INFINITY;
  Target target;
  if (tid == 0 && !p.parts) target = target_of(p, n, whole_row);

  auto collect = [&](float x, int i) {
    const int at = atomicAdd(&count, 1);
    if (at < kCands) cands[at] = order_key(x, begin + i);
  };
  auto take = [&](const uint4& q, int v) {
    float x[N];
    unpack16(q, x, T());
    sums.add(x, p.cap);
    if constexpr (TOP) {
      bool any = false;
#pragma unroll
      for (int i = 0; i < N; ++i) any |= !(x[i] <= bound);
      if (any)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (!(x[i] <= bound)) collect(x[i], v * N + i);
    }
  };

  // f(x, index) of every element
  auto each = [&](auto f) {
    for (int v = tid; v < whole; v += kThreads) {
      float x[N];
      unpack16(load_vec(row + (int64_t)v * N), x, T());
#pragma unroll
      for (int i = 0; i < N; ++i) f(x[i], v * N + i);
    }
    if (tid < V - whole * N) f(io_traits<T>::load(row + whole * N + tid), whole * N + tid);
  };

  // collects anew, what is not below `low`
  auto collect_from = [&](uint64_t low) {
    if (tid == 0) count = 0;
    __syncthreads();
    each([&](float x, int i) {
      if (order_key(x, begin + i) >= low) collect(x, i);
    });
    __syncthreads();
  };

  int v = tid;
  if constexpr (TOP) {
    if (tid < kGroups) groups[tid] = 0;
    if (tid == 0) count = 0;
    __syncthreads();
    uint4 q[kFirst];
#pragma unroll
    for (int j = 0; j < kFirst; ++j)
      if (v + j * kThreads < whole) q[j] = load_vec(row + (int64_t)(v + j * kThreads) * N);
    float top[kFirst], best = -INFINITY;  // of each vector (NaN if it holds one)
#pragma unroll
    for (int j = 0; j < kFirst; ++j)
      if (v + j * kThreads < whole) {
        float x[N];
        unpack16(q[j], x, T());
        sums.add(x, p.cap);
        top[j] = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top[j] = __builtin_elementwise_maximum(top[j], x[i]);
        best = __builtin_elementwise_maximum(best, top[j]);
      }
    // the first place of the largest (of a NaN some place behind all: a lower bound)
    int at = 0x7fffffff - lane - begin;
#pragma unroll
    for (int j = kFirst - 1; j >= 0; --j)
      if (v + j * kThreads < whole && top[j] == best) {
        float x[N];
        unpack16(q[j], x, T());
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
          if (x[i] == best) at = (v + j * kThreads) * N + i;
      }
    if (v < whole) atomicMax(&groups[lane], (unsigned long long)order_key(best, begin + at));
    __syncthreads();
    const uint64_t key = kth_of_lanes(groups[lane], p.top_k);
    // (fewer than top_k groups: the piece has few elements, and all are collected)
    bound = key == 0 ? NAN : key_value(key);
#pragma unroll
    for (int j = 0; j < kFirst; ++j)
      if (v + j * kThreads < whole && !(top[j] < bound)) {
        float x[N];
        unpack16(q[j], x, T());
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int at = (v + j * kThreads) * N + i;
          if (order_key(x[i], begin + at) >= key) collect(x[i], at);
        }
      }
    v += kFirst * kThreads;
  }
  for (; v < whole; v += kAhead * kThreads) {
    uint4 q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (v + j * kThreads < whole) q[j] = load_vec(row + (int64_t)(v + j * kThreads) * N);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (v + j * kThreads < whole) take(q[j], v + j * kThreads);
  }
  if (tid < V - whole * N) {
    const float x[1] = {io_traits<T>::load(row + whole * N + tid)};
    sums.add(x, p.cap);
    if (TOP && !(x[0] <= bound)) collect(x[0], whole * N + tid);
  }

  // join the threads' sums
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    sums.join(__shfl_xor(sums.m, d), __shfl_xor(sums.s, d), __shfl_xor(sums.a, d));
  if (lane == 0) {
    lds_sums[tid >> 6][0] = sums.m;
    lds_sums[tid >> 6][1] = sums.s;
    lds_sums[tid >> 6][2] = sums.a;
  }
  __syncthreads();
  sums = Sums<CAP>();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sums.join(lds_sums[w][0], lds_sums[w][1], lds_sums[w][2]);
  const int64_t part = n * p.pieces + blockIdx.y;
  float lse = 0.0f, entropy;
  if (p.parts) {
    if (tid < 3) p.part_sums[part * 3 + tid] = tid == 0 ? sums.m : tid == 1 ? sums.s : sums.a;
  } else {
    row_results(sums, p.cap, lse, entropy);
    if (tid == 0) store_row<CAP>(p, n, target, lse, entropy);
  }

  if constexpr (TOP) {
    int have = count;
    if (have > kCands) {
      for (int e = tid; e < kCands; e += kThreads) {
        const uint64_t mine = cands[e];
        int above = 0;
        for (int j = 0; j < kCands; ++j) above += cands[j] > mine;
        if (above == p.top_k - 1) bound_lds = mine;
      }
      __syncthreads();
      collect_from(bound_lds);
      have = count;
      __syncthreads();
    }
    if (have > kCands) {
      // keys below `low` are out; it has its digits above `shift`, and `above` of the keys are
      // greater in those
      uint64_t low = 0;
      int above = 0;
      int* digits = reinterpret_cast<int*>(cands);
      for (int shift = 56; shift >= 0 && have > kCands; shift -= 8) {
        digits[tid] = 0;
        __syncthreads();
        each([&](float x, int i) {
          const uint64_t key = order_key(x, begin + i);
          if (key >> shift >> 8 != low >> shift >> 8) return;
          // (lanes of one digit count as one: equal logits, and the digits above those that
          // differ, would queue for the same word)
          const int digit = (int)(key >> shift) & 255;
          const uint64_t here = __ballot(1);
          if (__ballot(digit == __builtin_amdgcn_readfirstlane(digit)) != here)
            atomicAdd(&digits[digit], 1);
          else if (lane == __builtin_ctzll(here))
            atomicAdd(&digits[digit], __builtin_popcountll(here));
        });
        __syncthreads();
        // the greatest digit that leaves top_k keys, four digits to a lane
        if (tid < 64) {
          int c[4], sum = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += c[e] = digits[255 - 4 * tid - e];
          int before = sum;
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(before, d);
            if (tid >= d) before += y;
          }
          before += above - sum;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (before < p.top_k && before + c[e] >= p.top_k) {
              bound_lds = low | (uint64_t)(255 - 4 * tid - e) << shift;
              above_lds = before;
              count = before + c[e];
            }
            before += c[e];
          }
        }
        __syncthreads();
        low = bound_lds;
        above = above_lds;
        have = count;
        __syncthreads();
      }
      collect_from(low);
      have = count;
    }
    for (int e = tid; e < have; e += kThreads) {
      const uint64_t mine = cands[e];
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < have; ++j) above += cands[j] > mine;
      if (above >= p.top_k) continue;
      if (p.parts) {
        p.part_keys[part * p.top_k + above] = mine;
      } else {
        p.top_ids[n * p.top_k + above] = key_index(mine);
        p.top_lp[n * p.top_k + above] = capped<CAP>(key_value(mine), p.cap) - lse;
      }
    }
    // (a last piece of fewer elements than alternatives)
    if (p.parts)
      for (int e = have + tid; e < p.top_k; e += kThreads) p.part_keys[part * p.top_k + e] = 0;
  }
}

constexpr int kPieces = 16;  // of a row, at most

constexpr int kJoinThreads = kPieces * kGroups;

// Joins a row's pieces: one workgroup, every piece's sums, and the best of the pieces'
// alternatives.  The k-th largest of the first few of every piece bounds the k-th largest of
// all from below; what is not under it, hardly more than k, is collected and ranked.
// (16 rows of 16 pieces with 20 alternatives: 3.1 us, with all ranked against all 5.7.)
template <typename T, Cap CAP>
__global__ void __launch_bounds__(kJoinThreads) logprobs_join_kernel(const LogpArgs p) {
  __shared__ unsigned long long cands[kJoinThreads];
  __shared__ unsigned long long bound;
  __shared__ int count;
  __shared__ float lse_lds;
  const int64_t n = blockIdx.x;
  const int tid = threadIdx.x, all = p.pieces * p.top_k;
  const uint64_t mine = tid < all ? p.part_keys[n * all + tid] : 0;
  if (tid < 64 && all > 0) {
    const int each = min(64 / p.pieces, p.top_k), piece = tid / each;
    const uint64_t key = piece < p.pieces
                             ? p.part_keys[n * all + piece * p.top_k + tid - piece * each] : 0;
    const uint64_t kth = kth_of_lanes(key, p.top_k);
    if (tid == 0) {
      bound = kth;
      count = 0;
    }
  }
  Target target;
  if (tid == 0) target = target_of(p, n, reinterpret_cast<const T*>(p.x) + n * p.xs);
  // (lanes past the pieces hold nothing)
  Sums<CAP> sums;
  const float* part = p.part_sums + (n * p.pieces + (tid & 63)) * 3;
  if ((tid & 63) < p.pieces) {
    sums.m = part[0];
    sums.s = part[1];
    sums.a = part[2];
  }
#pragma unroll
  for (int d = 1; d < kPieces; d <<= 1)
    sums.join(__shfl_xor(sums.m, d), __shfl_xor(sums.s, d), __shfl_xor(sums.a, d));
  if (tid == 0) {
    float lse, entropy;
    row_results(sums, p.cap, lse, entropy);
    store_row<CAP>(p, n, target, lse, entropy);
    lse_lds = lse;
  }
  if (all == 0) return;
  __syncthreads();
  // (0: no entry)
  if (mine != 0 && mine >= bound) cands[atomicAdd(&count, 1)] = mine;
  __syncthreads();
  const int have = count;
  if (tid >= have) return;
  const uint64_t key = cands[tid];
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < have; ++j) rank += cands[j] > key;
  if (rank < p.top_k) {
    p.top_ids[n * p.top_k + rank] = key_index(key);
    p.top_lp[n * p.top_k + rank] = capped<CAP>(key_value(key), p.cap) - lse_lds;
  }
}

// Pieces that a row is cut into: one for 512 rows and more, which fill the card; else up to
// 16, of 4,096 elements at least, towards 1,024 workgroups.
int row_pieces(int64_t N, int V) {
  if (N >= 512 || N <= 0) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({kPieces, (1024 + N - 1) / N, V / 4096}));
}

// (a multiple of 64 elements: pieces of an aligned row are aligned)
int piece_size(int V, int pieces) {
  return (int)std::min<int64_t>((((int64_t)V + pieces - 1) / pieces + 63) / 64 * 64, V);
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
  int piece;  // elements of a workgroup
};

// dx of an element, without the terms of a target or an alternative (extra).
template <Cap CAP>
struct Grad {
  float lse, total, ge, ent, cap, cap_scale;
  __device__ __forceinline__ float operator()(float x, float extra) const {
    float z = x, slope = 1.0f;
    if constexpr (CAP == kCap) {
      const float r = cap_r(x, cap_scale);
      z = fmaf(-2.0f * cap, r, cap);
      slope = 4.0f * r * (1.0f - r);
    } else if constexpr (CAP == kWideCap) {
      z = wide_capped(x, cap);
      const float t = z / cap;
      slope = fmaf(-t, t, 1.0f);
    }
    const float lp = z - lse, e = __builtin_amdgcn_exp2f(lp * kLog2e);
    // (an entry without probability has none, however low its log and large the gradient)
    const float d = -e * fmaf(ge, fmaxf(lp, -1000.0f) + ent, total);
    return (d + extra) * slope;
  }
};

// kGradThreads: 1,024 for pieces of 64 KiB and more, so that fewer are read and written side by
// side (4,096 rows of 50,257 bfloat16 logits, forward and gradient, 275 us with 256, 265 with
// 512, 257 with 1,024; the gradient of 2,000 rows of float32 171 and 145), else 256 (2,000 rows
// of bfloat16, pieces of 40 KiB, 86 and 89; 4,096 of 1,000 logits 7 and 13).
template <typename T, Cap CAP, int kGradThreads>
__global__ void __launch_bounds__(kGradThreads) logprobs_backward_kernel(const LogpGradArgs p) {
  constexpr int N = io_traits<T>::kVec, kAhead = 2;
  const int64_t n = blockIdx.y;
  const int begin = blockIdx.x * p.piece, end = min(p.V - begin, p.piece) + begin;
  const T* x = reinterpret_cast<const T*>(p.x) + n * p.xs;
  T* gx = reinterpret_cast<T*>(p.gx) + n * p.gs;
  const int tid = threadIdx.x;
  const int64_t target = p.targets[n];
  const bool given = target >= 0 && target < p.V;
  const float g = given && p.g_lp != nullptr ? p.g_lp[n] : 0.0f;
  const int k = p.g_top != nullptr ? p.top_k : 0;
  Grad<CAP> grad;
  grad.lse = p.lse[n];
  grad.ge = p.g_ent != nullptr ? p.g_ent[n] : 0.0f;
  grad.ent = p.g_ent != nullptr ? p.entropy[n] : 0.0f;
  grad.cap = p.cap;
  grad.cap_scale = CAP == kCap ? cap_scale_of(p.cap) : 0.0f;
  grad.total = g;
  for (int i = 0; i < k; ++i) grad.total += p.g_top[n * p.top_k + i];

  const int whole = (end - begin) / N;
  for (int v = tid; v < whole; v += kAhead * kGradThreads) {
    uint4 q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (v + j * kGradThreads < whole)
        q[j] = load_vec(x + begin + (int64_t)(v + j * kGradThreads) * N);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (v + j * kGradThreads < whole) {
        float f[N];
        unpack16(q[j], f, T());
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = grad(f[i], 0.0f);
        uint4 o;
        if constexpr (sizeof(T) == 2)
          o = make_uint4(cvt_pk_bf16(f[0], f[1]), cvt_pk_bf16(f[2], f[3]), cvt_pk_bf16(f[4], f[5]),
                         cvt_pk_bf16(f[6], f[7]));
        else
          o = pack16(f, T());
        __builtin_memcpy(gx + begin + (int64_t)(v + j * kGradThreads) * N, &o, 16);
      }
  }
  if (tid < end - begin - whole * N) {
    const int j = begin + whole * N + tid;
    io_traits<T>::store(gx + j, grad(io_traits<T>::load(x + j), 0.0f));
  }
  __syncthreads();
  // the target's and the alternatives' elements again (thread k: a target that is none)
  if (tid <= k) {
    int64_t j = tid < k ? p.top_ids[n * p.top_k + tid] : given ? target : -1;
    float extra = tid < k ? p.g_top[n * p.top_k + tid] + (j == target ? g : 0.0f) : g;
    if (tid == k)
      for (int i = 0; i < k; ++i)
        if (p.top_ids[n * p.top_k + i] == j) j = -1;
    if (j >= begin && j < end)
      io_traits<T>::store(gx + j, grad(io_traits<T>::load(x + j), extra));
  }
}

template <Cap CAP>
using cap_type = std::integral_constant<Cap, CAP>;

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

int logprobs_pieces(int64_t N, int V) {
  const int piece = piece_size(V, row_pieces(N, V));
  return (int)(((int64_t)V + piece - 1) / piece);
}

int logprobs_parts(int dtype, const void* x, int64_t row_stride, const uint8_t* skip,
                   float* part_sums, uint64_t* part_keys, int64_t N, int V, int top_k,
                   float softcap, hipStream_t stream) {
  LogpArgs a{x, row_stride, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, V, top_k,
             softcap, piece_size(V, row_pieces(N, V)), logprobs_pieces(N, V), true, skip, part_sums,
             part_keys};
  const dim3 grid((unsigned)N, a.pieces);
  auto launch = [&](auto type) {
    using T = decltype(type);
    auto by_cap = [&](auto cap) {
      hipLaunchKernelGGL((logprobs_forward_kernel<T, decltype(cap)::value, true>), grid,
                         dim3(kThreads), 0, stream, a);
    };
    // (float32 z of large caps are off by 2^-22 of themselves and more, each in its own way: of two
    // beams with one likely continuation each that would decide)
    switch (exact_cap_of(softcap)) {
      case kNoCap: return by_cap(cap_type<kNoCap>());
      case kCap: return by_cap(cap_type<kCap>());
      case kCap64: return by_cap(cap_type<kCap64>());
      default: return by_cap(cap_type<kTanh64>());
    }
  };
  if (dtype == LTV_DTYPE_F32) launch(float()); else launch(bf16_t());
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}

}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_token_logprobs_workspace_size(int64_t N, int V, int top_k) {
  if (N <= 0 || V <= 0 || top_k < 0 || row_pieces(N, V) == 1) return 0;
  return (size_t)N * row_pieces(N, V) * (top_k * sizeof(uint64_t) + 3 * sizeof(float));
}

extern "C" int ltv_token_logprobs_forward(int dtype, const void* logits, int64_t row_stride,
                                          const int64_t* targets, float* logprobs, float* entropy,
                                          float* lse, float* top_logprobs, int64_t* top_ids,
                                          void* workspace, size_t workspace_bytes, int64_t N,
                                          int V, int top_k, float softcap, void* stream) {
  const int bad = check_rows(dtype, logits, row_stride, targets, N, V, top_k, softcap);
  if (bad != LTV_OK) return bad;
  if (N == 0) return LTV_OK;
  LTV_REQUIRE(logprobs && (top_k == 0 || (top_logprobs && top_ids)), LTV_ERR_INVALID_ARG,
              "null output");
  const int pieces = row_pieces(N, V);
  LTV_REQUIRE(workspace_bytes >= ltv_token_logprobs_workspace_size(N, V, top_k) &&
                  (pieces == 1 || (workspace && aligned16(workspace))),
              LTV_ERR_WORKSPACE, "workspace too small");
  uint64_t* keys = reinterpret_cast<uint64_t*>(workspace);
  const int piece = piece_size(V, pieces);
  LogpArgs a{logits, row_stride, targets, logprobs, entropy, lse, top_logprobs, top_ids,
                   V, top_k, softcap, piece, (int)(((int64_t)V + piece - 1) / piece), pieces > 1,
                   nullptr, reinterpret_cast<float*>(keys + N * pieces * top_k), keys};
  const hipStream_t st = (hipStream_t)stream;
  // (a launch has less than 2^32 threads along an axis; so many rows are not cut)
  constexpr int64_t kMostRows = int64_t(1) << 23;
  auto launch = [&](auto type, auto cap) -> int {
    using T = decltype(type);
    constexpr Cap C = decltype(cap)::value;
    for (int64_t n0 = 0; n0 < N; n0 += kMostRows) {
      const int64_t m = std::min(kMostRows, N - n0);
      const dim3 grid((unsigned)m, a.pieces);
      if (top_k > 0)
        hipLaunchKernelGGL((logprobs_forward_kernel<T, C, true>), grid, dim3(kThreads), 0, st, a);
      else
        hipLaunchKernelGGL((logprobs_forward_kernel<T, C, false>), grid, dim3(kThreads), 0, st,
                           a);
      LTV_LAUNCH_CHECK();
      if (n0 + m == N) break;
      a.x = (const T*)a.x + m * row_stride;
      a.targets += m;
      a.logprobs += m;
      a.entropy = a.entropy ? a.entropy + m : nullptr;
      a.lse = a.lse ? a.lse + m : nullptr;
      a.top_lp = a.top_lp ? a.top_lp + m * top_k : nullptr;
      a.top_ids = a.top_ids ? a.top_ids + m * top_k : nullptr;
    }
    if (a.pieces > 1) {
      hipLaunchKernelGGL((logprobs_join_kernel<T, C>), dim3((unsigned)N), dim3(kJoinThreads),
                         0, st, a);
      LTV_LAUNCH_CHECK();
    }
    return LTV_OK;
  };
  auto by_cap = [&](auto type) {
    if (softcap > kMostCap) return launch(type, cap_type<kWideCap>());
    return softcap > 0.0f ? launch(type, cap_type<kCap>()) : launch(type, cap_type<kNoCap>());
  };
  return dtype == LTV_DTYPE_F32 ? by_cap(float()) : by_cap(bf16_t());
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
  // rows are cut into pieces, of 4,096 elements at least, until there are 4,096 of them
  const int64_t want = std::max<int64_t>(1, (4096 + N - 1) / N);
  const int piece = (int)std::min<int64_t>(
      std::max<int64_t>(4096, ((V + want - 1) / want + 4095) / 4096 * 4096), 1 << 30);
  LogpGradArgs a{logits, row_stride, targets, lse, entropy, top_ids, g_logprobs, g_entropy,
                 g_top, grad_logits, grad_row_stride, V, top_k, softcap, piece};
  const hipStream_t st = (hipStream_t)stream;
  // (the grid's second axis ends at 65,535)
  for (int64_t n0 = 0; n0 < N; n0 += 65535) {
    const dim3 grid((unsigned)(((int64_t)V + piece - 1) / piece), (unsigned)std::min<int64_t>(65535, N - n0));
    auto launch = [&](auto type, auto cap) {
      using T = decltype(type);
      constexpr Cap C = decltype(cap)::value;
      if ((int64_t)std::min(piece, V) * (int)sizeof(T) >= 65536)
        hipLaunchKernelGGL((logprobs_backward_kernel<T, C, 1024>), grid, dim3(1024), 0, st, a);
      else
        hipLaunchKernelGGL((logprobs_backward_kernel<T, C, 256>), grid, dim3(256), 0, st, a);
    };
    auto by_cap = [&](auto type) {
      if (softcap > kMostCap) launch(type, cap_type<kWideCap>());
      else if (softcap > 0.0f) launch(type, cap_type<kCap>());
      else launch(type, cap_type<kNoCap>());
    };
    if (dtype == LTV_DTYPE_F32) by_cap(float()); else by_cap(bf16_t());
    LTV_LAUNCH_CHECK();
    const int64_t m = grid.y;
    const int es = dtype == LTV_DTYPE_F32 ? 4 : 2;
    a.x = (const char*)a.x + m * row_stride * es;
    a.gx = (char*)a.gx + m * grad_row_stride * es;
    a.targets += m;
    a.lse += m;
    a.entropy = a.entropy ? a.entropy + m : nullptr;
    a.g_lp = a.g_lp ? a.g_lp + m : nullptr;
    a.g_ent = a.g_ent ? a.g_ent + m : nullptr;
    a.top_ids = a.top_ids ? a.top_ids + m * top_k : nullptr;
    a.g_top = a.g_top ? a.g_top + m * top_k : nullptr;
  }
  return LTV_OK;
}
