// A search's selection: the k best continuations of a prompt's beams.
//
//   of (beam b, token v):  scores[b] + z[b, v] - lse[b],  z = c tanh(x / c)  (or x)
//
// The logits are read once, by the pass of the token log probabilities: it leaves, of each piece
// of a row, the sum of its exponentials and its k largest logits, more than which no beam can
// have among the best.  One workgroup for each prompt joins them: a wavefront takes a beam's
// pieces, and then the beams' candidates are ranked, each by counting those before it.
//
// A score decides which of two beams goes on, so scores are float64, and so is what they are made
// of as far as it may matter: a candidate's z, the joined sums and their logarithm, and of caps
// past 64 every z of the pass (a float32 one is off by more than the log probability of a likely
// token).  Of smaller caps the exponentials of the pass are off by some roundings of the cap, all
// alike in size.  Of a few logits that have most of the sum that would show in lse, so with a cap
// the candidates' terms (the largest there are) are taken out of the sum as they went in and put
// back exactly.  What is left is the float32 sum's: terms and additions off by some 2^-24 each.
//
// Bounded by the pass over the logits: 384 beams' rows of 50,257 bfloat16 (39 MB) 22 us, 1.8 TB/s --
// at that length it is the pass's start, its bound for the candidates and its join within a
// workgroup, three pieces to a row (2, 3, 6 and 11 pieces: 20.5, 21, 24 and 29 us).  The joining
// is latency: 7 us for 48 prompts of 8 beams each, 5 for one of 4.
#include <algorithm>

#include "../../include/nanochat_decoding_amd.h"
#include "ltv_logprobs.hpp"

namespace ltv {
namespace {

constexpr int kMostBeams = 1024;  // times candidates of each
constexpr int kMostPieces = 16;   // of a row

struct BeamArgs {
  const float* sums;     // (G * B, pieces, 3)
  const uint64_t* keys;  // (G * B, pieces, n)
  const float* scores;
  const uint8_t* finished;
  float* out_scores;
  int64_t* parents;
  int64_t* tokens;
  int B, pieces, n, k;  // n: candidates of a beam
  float cap;
};

// Larger scores first, NaN above all.
__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return x != x ? ~0ull : u >> 63 ? ~u : u | 1ull << 63;
}

// What a wavefront's lanes wrote to LDS is there for its others.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ double wave_sum(double x) {
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

template <Cap CAP>
__global__ void beam_kernel(const BeamArgs a) {
  extern __shared__ uint64_t lds[];
  const int entries = a.B * a.n, all = a.pieces * a.n;
  uint64_t* order = lds;                                  // (B, n) scores' keys
  double* score = reinterpret_cast<double*>(lds + entries);  // (B, n)
  int* token = reinterpret_cast<int*>(lds + 2 * entries);    // (B, n)
  int* before = token + entries;                          // (B, n)
  uint64_t* mine = lds + 3 * entries;                     // (waves, pieces * n), pieces > 1
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  mine += wave * all;
  const int64_t g = blockIdx.x;
  for (int b = wave; b < a.B; b += waves) {
    const int64_t row = g * a.B + b;
    // (all on their way at once, also what a finished beam has no use for)
    const uint64_t* keys = a.keys + row * all;
    const float* part = a.sums + (row * a.pieces + lane) * 3;
    const uint64_t first = lane < all ? keys[lane] : 0;
    double m = 0.0, sum = 0.0;
    if (lane < a.pieces) {
      m = part[0];
      sum = part[1];
    }
    const double s = a.scores[row];
    const bool finished = a.finished != nullptr && a.finished[row] != 0;
    for (int r = lane; r < a.n; r += 64) before[b * a.n + r] = 0;
    if (finished) {
      for (int r = lane; r < a.n; r += 64) {
        const double x = r == 0 ? s : -INFINITY;
        order[b * a.n + r] = score_key(x);
        score[b * a.n + r] = x;
        token[b * a.n + r] = -1;
      }
      continue;
    }
    // the n largest of the pieces' keys, in order, into this beam's part of `order`
    if (a.pieces == 1) {
      if (lane < a.n) order[b * a.n + lane] = first;
    } else if (all <= 64) {
      int rank = 0;
      for (int j = 0; j < all; ++j) rank += of_lane(first, j) > first;
      if (first != 0 && rank < a.n) order[b * a.n + rank] = first;
    } else {
      // (the n-th of the first few of every piece is a bound)
      const int each = min(64 / a.pieces, a.n), piece = lane / each;
      const uint64_t head = piece < a.pieces ? keys[piece * a.n + lane - piece * each] : 0;
      const uint64_t bound = kth_of_lanes(head, a.n);
      int have = 0;
      for (int i0 = 0; i0 < all; i0 += 64) {
        const uint64_t key = i0 == 0 ? first : i0 + lane < all ? keys[i0 + lane] : 0;
        const bool in = key != 0 && key >= bound;
        const uint64_t who = __ballot(in);
        if (in) mine[have + __builtin_popcountll(who & ((1ull << lane) - 1))] = key;
        have += __builtin_popcountll(who);
      }
      wave_sync();
      for (int i = lane; i < have; i += 64) {
        const uint64_t key = mine[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < have; ++j) rank += mine[j] > key;
        if (rank < a.n) order[b * a.n + rank] = key;
      }
    }
    wave_sync();
    // the row's sums
    if constexpr (CAP != kCap) {
      double top = lane < a.pieces ? m : -INFINITY;
      for (int d = 1; d < kMostPieces; d <<= 1) top = fmax(top, __shfl_xor(top, d));
      // (a piece of -inf alone has the sum 0; a NaN in a sum stays)
      if (lane < a.pieces && m != -INFINITY) sum *= exp(m - top);
      m = __shfl(top, 0);
    } else {
      m = 0.0;
    }
    // the candidates' z, and the exact terms in place of the pass's (n is at most 64; without a cap
    // the largest is 1 in both)
    double z = 0.0;
    if (lane < a.n) {
      const uint64_t key = order[b * a.n + lane];
      const float x = key_value(key);
      z = capped64<CAP>(x, a.cap);
      if constexpr (CAP == kCap)
        sum += exp(z) - (double)cap_exp(cap_r(x, cap_scale_of(a.cap)), a.cap);
      if constexpr (CAP == kCap64 || CAP == kTanh64)
        sum += exp(z - m) - (double)below_exp(z, (float)m);
      token[b * a.n + lane] = key_index(key);
    }
    sum = wave_sum(sum);
    if (lane < a.n) {
      const double lse = m + log(sum);
      const double x = s == -INFINITY || z == -INFINITY ? -INFINITY : s + (z - lse);
      score[b * a.n + lane] = x;
      order[b * a.n + lane] = score_key(x);
    }
  }
  __syncthreads();
  // By score, beam and place in the beam: how many are before each, counted by all threads.
  const int shares = max(1, (int)blockDim.x / entries);
  for (int u = threadIdx.x; u < entries * shares; u += blockDim.x) {
    const int share = u / entries, i = u - share * entries;
    const uint64_t key = order[i];
    int rank = 0;
#pragma unroll 4
    for (int j = share; j < entries; j += shares) {
      const uint64_t other = order[j];
      rank += other > key || (other == key && j < i);
    }
    if (shares > 1) atomicAdd(&before[i], rank); else before[i] = rank;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < entries; i += blockDim.x) {
    const int rank = before[i];
    if (rank >= a.k) continue;
    const int64_t at = g * a.k + rank;
    a.out_scores[at] = (float)score[i];
    a.parents[at] = i / a.n;
    a.tokens[at] = token[i];
  }
}

size_t beam_lds(int B, int n, int pieces, int waves) {
  return ((size_t)3 * B * n + (pieces > 1 ? (size_t)waves * pieces * n : 0)) * sizeof(uint64_t);
}

}  // namespace
}  // namespace ltv

using namespace ltv;

extern "C" size_t ltv_beam_select_workspace_size(int64_t groups, int beams, int V, int k) {
  if (groups <= 0 || beams <= 0 || V <= 0 || k <= 0) return 0;
  const int64_t N = groups * beams;
  return (size_t)N * logprobs_pieces(N, V) *
         (std::min(k, V) * sizeof(uint64_t) + 3 * sizeof(float));
}

extern "C" int ltv_beam_select(int dtype, const void* logits, int64_t row_stride,
                               const float* scores, const uint8_t* finished, float* out_scores,
                               int64_t* parents, int64_t* tokens, void* workspace,
                               size_t workspace_bytes, int64_t groups, int beams, int V, int k,
                               float softcap, void* stream) {
  LTV_REQUIRE(dtype == LTV_DTYPE_F32 || dtype == LTV_DTYPE_BF16, LTV_ERR_INVALID_ARG,
              "unknown dtype %d", dtype);
  LTV_REQUIRE(groups >= 0 && beams > 0 && V > 0 && k > 0 && (int64_t)beams * V >= k,
              LTV_ERR_INVALID_ARG, "bad shape (groups=%lld beams=%d V=%d k=%d)",
              (long long)groups, beams, V, k);
  LTV_REQUIRE(softcap >= 0.0f && softcap < INFINITY, LTV_ERR_INVALID_ARG,
              "softcap must be finite and not negative");
  const int n = std::min(k, V);
  LTV_REQUIRE(n <= 64 && (int64_t)beams * n <= kMostBeams, LTV_ERR_UNSUPPORTED,
              "at most 64 continuations of a beam and %d of all (beams=%d k=%d)", kMostBeams, beams,
              k);
  LTV_REQUIRE(groups <= (int64_t(1) << 20) / beams, LTV_ERR_UNSUPPORTED, "too many rows");
  if (groups == 0) return LTV_OK;
  LTV_REQUIRE(logits && scores && out_scores && parents && tokens, LTV_ERR_INVALID_ARG,
              "null pointer");
  LTV_REQUIRE(workspace && aligned16(workspace) &&
                  workspace_bytes >= ltv_beam_select_workspace_size(groups, beams, V, k),
              LTV_ERR_WORKSPACE, "workspace too small");
  const int64_t N = groups * beams;
  const int pieces = logprobs_pieces(N, V);
  uint64_t* keys = reinterpret_cast<uint64_t*>(workspace);
  float* sums = reinterpret_cast<float*>(keys + N * pieces * n);
  const hipStream_t st = (hipStream_t)stream;
  const int rc = logprobs_parts(dtype, logits, row_stride, finished, sums, keys, N, V, n, softcap,
                                st);
  if (rc != LTV_OK) return rc;
  const BeamArgs a{sums, keys, scores, finished, out_scores, parents, tokens, beams, pieces, n, k,
                   softcap};
  // (as many wavefronts as there are beams, or as the LDS that a launch may have holds)
  int waves = std::min(16, beams);
  while (waves > 1 && beam_lds(beams, n, pieces, waves) > 60000) --waves;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(64 * waves),
                       beam_lds(beams, n, pieces, waves), st, a);
  };
  switch (exact_cap_of(softcap)) {
    case kNoCap: launch(beam_kernel<kNoCap>); break;
    case kCap: launch(beam_kernel<kCap>); break;
    case kCap64: launch(beam_kernel<kCap64>); break;
    default: launch(beam_kernel<kTanh64>); break;
  }
  LTV_LAUNCH_CHECK();
  return LTV_OK;
}
