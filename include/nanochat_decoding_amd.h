/*
 * nanochat_decoding_amd.h -- C ABI of the MI355X (gfx950) operators of a decoding
 * step beside those of nanochat_serving_amd.h: rotation of new tokens on their way
 * into a paged cache, caches held in 4 bits, sequences that change places, and a
 * search's selection.  Part of libnanochat_filter_amd.so.
 *
 * The conventions are those of nanochat_serving_amd.h: raw device pointers, int64
 * element strides, a dtype code, a hipStream_t; a call only enqueues work on that
 * stream, allocates nothing and returns LTV_OK or an LTV_ERR_* code with the message
 * in ltv_last_error().  What is read on the device is checked there.
 *
 * Pages in 4 bits (LTV_PAGES_FP4): uint8 arrays (P, NKVH, page, D / 2 + D / 32) whose
 * last two axes are one dense block, D and the page size multiples of 32 and 16, pages
 * and heads multiples of 16 bytes apart, 16-byte aligned.  Of a page and head, the block is
 *   codes  (page, D / 2)  : token by token, channel 2 i in the low half of byte i
 *   scales (D / 32, page) : one byte for 32 channels of a token
 * and stands for the values  m * 2^(scale - 127),  m the code's: its low three bits
 * give 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the fourth the sign.  Scales are 2 to 252 (all
 * values are normal bfloat16 numbers), or 255: the 32 channels are NaN.
 * Values x are held with the scale of the smallest power of two s by which no |x| is
 * larger than 7 (scale 2 to 252: far smaller or larger values become 0 or the largest)
 * and the nearest code of x / s, ties to the even code, 6 for what is beyond; 32 channels
 * with an infinity or NaN among them are NaN.
 */
#ifndef NANOCHAT_DECODING_AMD_H
#define NANOCHAT_DECODING_AMD_H

#include "nanochat_serving_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this ABI (bumped on any signature change or addition): 1. */
int ltv_decoding_abi_version(void);

#define LTV_PAGES_VALUES 0 /* in the tokens' dtype */
#define LTV_PAGES_FP4 1

/* ------------------------------------------------------------------------
 * Rotates the new tokens' queries and keys by their positions, normalises them, and
 * writes the keys and values into their pages:
 *   y[i]         = x[i] cos[pos, i] + x[i + D / 2] sin[pos, i]        0 <= i < D / 2
 *   y[i + D / 2] = x[i + D / 2] cos[pos, i] - x[i] sin[pos, i]
 *   norm_eps >= 0: y / sqrt(mean y^2 + norm_eps);  norm_eps < 0: y
 * q_out holds the queries' (of a token at a negative position: 0), the pages the keys';
 * values go into the pages as they are.  Computed in float64 and rounded once.
 *
 * q, k, v, q_out: token rows (heads, D), strides (sequence, token, head), last stride 1,
 * any alignment.  cos, sin: (positions, D / 2) of table_dtype, row strides in elements,
 * last stride 1; positions >= table_width * page_size.  k_page_strides, v_page_strides:
 * (page, head, token), of LTV_PAGES_FP4 in bytes with the token's D / 2 + D / 32.
 * D a multiple of 8, at most 128 (LTV_PAGES_FP4: of 32).  B <= 65,535; total * heads < 2^27.
 * ---------------------------------------------------------------------- */
int ltv_paged_rotary_append(int dtype, const void* q, const int64_t q_strides[3], const void* k,
                            const int64_t k_strides[3], const void* v, const int64_t v_strides[3],
                            const void* cos, int64_t cos_stride, const void* sin,
                            int64_t sin_stride, int table_dtype, int64_t positions,
                            double norm_eps, void* q_out, const int64_t q_out_strides[3],
                            void* k_pages, const int64_t k_page_strides[3], void* v_pages,
                            const int64_t v_page_strides[3], int page_format,
                            const ltv_paged_batch* batch, int NH, int NKVH, int D, void* stream);

/* Writes the new tokens' keys and values into 4-bit pages; arguments as of
 * ltv_paged_cache_append, limits as above. */
int ltv_paged_cache_append_fp4(int dtype, const void* k, const int64_t k_strides[3],
                               const void* v, const int64_t v_strides[3], void* k_pages,
                               const int64_t k_page_strides[3], void* v_pages,
                               const int64_t v_page_strides[3], const ltv_paged_batch* batch,
                               int NKVH, int D, void* stream);

/* What the pages hold of the new tokens: k_out, v_out (total, NKVH, D) of dtype, 16-byte
 * aligned and contiguous, every row written (0: a token at a negative position or of no
 * page, or, with starts, a row of no sequence).  LTV_PAGES_VALUES: dtype is the pages'. */
int ltv_paged_cache_read(int dtype, int page_format, const void* k_pages,
                         const int64_t k_page_strides[3], const void* v_pages,
                         const int64_t v_page_strides[3], const ltv_paged_batch* batch,
                         void* k_out, void* v_out, int NKVH, int D, void* stream);

/* ltv_paged_attention over 4-bit pages: the same sums over the values that the pages stand
 * for, q and out of dtype.  D 32, 64, 96 or 128; page strides in bytes, pages of a layer
 * within 32 GiB.  max_len is a hint that chooses launch shapes and no roundings.  Keys and values
 * that a token does not attend to never reach its output. */
size_t ltv_paged_attention_fp4_workspace_size(int dtype, const ltv_paged_batch* batch, int NH,
                                              int NKVH, int D, int max_len);
int ltv_paged_attention_fp4(int dtype, const void* q, const int64_t q_strides[3],
                            const void* k_pages, const int64_t k_page_strides[3],
                            const void* v_pages, const int64_t v_page_strides[3],
                            const ltv_paged_batch* batch, void* out, const int64_t out_strides[3],
                            float* lse, void* workspace, size_t workspace_bytes, int NH, int NKVH,
                            int D, int max_len, float scale, void* stream);

/* Slot slots[i] becomes what slot src[i] holds before the call, all n entries at once (a
 * slot may be named in src several times, and in both); pages are shared, and what is held
 * no longer is let go.  slots are distinct; an entry with a slot outside [0, num_slots) does
 * nothing.  n <= 65,535.  workspace: ltv_paged_cache_reorder_workspace_size bytes, 16-byte
 * aligned. */
size_t ltv_paged_cache_reorder_workspace_size(int n, int table_width);
int ltv_paged_cache_reorder(const ltv_page_state* state, const int32_t* slots, const int32_t* src,
                            int n, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * A search's selection: of each of `groups` prompts with `beams` beams, the k best
 * continuations over all beams and tokens.  logits x (groups * beams, V), row stride
 * row_stride, last stride 1; scores (groups, beams) float32, contiguous, the beams' own.
 *   score(b, v) = scores[b] + z[b, v] - log sum_w exp z[b, w],  z = softcap tanh(x / softcap)
 *                 (softcap 0: z = x);  -inf where scores[b] or z[b, v] is
 * in descending order (NaN above all); equal ones by beam, then by logit as top_ids of
 * ltv_token_logprobs_forward.  A beam with finished[b] != 0 (finished may be NULL) has one
 * continuation, itself, with its score and the token -1, and then min(k, V) - 1 with the
 * score -inf and the token -1; its logits are not read.
 *   out_scores (groups, k) float32, parents and tokens (groups, k): beam and token
 * k <= beams * V; min(k, V) <= 64 and beams * min(k, V) <= 1024; groups * beams <= 2^20.
 * Scores are compared in float64; the rows' sums are float32, off by some 2^-24 of them and, of
 * caps up to 64, by some 2^-23 of the cap.  workspace: ltv_beam_select_workspace_size bytes, 16-byte
 * aligned.
 * ---------------------------------------------------------------------- */
size_t ltv_beam_select_workspace_size(int64_t groups, int beams, int V, int k);
int ltv_beam_select(int dtype, const void* logits, int64_t row_stride, const float* scores,
                    const uint8_t* finished, float* out_scores, int64_t* parents, int64_t* tokens,
                    void* workspace, size_t workspace_bytes, int64_t groups, int beams, int V,
                    int k, float softcap, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOCHAT_DECODING_AMD_H */
