/*
 * nanochat_serving_amd.h -- C ABI of the MI355X (gfx950) serving operators: a
 * paged cache of attention keys and values, attention of new tokens over it,
 * and log probabilities of given tokens.  Part of libnanochat_filter_amd.so.
 *
 * The conventions are those of nanochat_filter_amd.h: raw device pointers,
 * int64 element strides, a dtype code, a hipStream_t; a call only enqueues work
 * on that stream, allocates nothing and returns LTV_OK or an LTV_ERR_* code with
 * the message in ltv_last_error().
 *
 * A paged cache (one layer of it):
 *   k_pages, v_pages : (P, NKVH, page, D), last stride 1, 16-byte aligned
 *   page_table       : (S, W) int32, row stride table_stride: the pages of slot s in
 *                      the order of its tokens; an id outside [0, P) holds no tokens
 *   seq_lens         : (S) int32, tokens of each slot
 *   ref_counts       : (P) int32, how many slots hold a page; 0: free
 * Lengths, page ids, slots and starts are read on the device, so a step can be
 * captured in a HIP graph and replayed while they change; every index derived
 * from them is checked there.
 */
#ifndef NANOCHAT_SERVING_AMD_H
#define NANOCHAT_SERVING_AMD_H

#include "nanochat_filter_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this ABI (bumped on any signature change or addition): 1. */
int ltv_serving_abi_version(void);

/* ------------------------------------------------------------------------
 * The sequences of one call and their new tokens.
 *
 * Sequence i (0 <= i < B) is slot slots[i] (slots NULL: slot i) and has n_i new
 * tokens, the last n_i of its seq_lens[slot] tokens:
 *   starts NULL: n_i = T, token t of sequence i at row (i, t) of the (B, T, ...)
 *                tensors;
 *   else         n_i = starts[i + 1] - starts[i], token t at row starts[i] + t of
 *                the (total, ...) tensors (starts: B + 1 int32, ascending); T is
 *                the largest n_i that is expected (a hint: more are computed too).
 * Token t is at position seq_lens[slot] - n_i + t; at a negative position it is
 * no token (appended nowhere, attends to nothing).  A slot outside [0, num_slots)
 * is an empty sequence.
 *
 * Limits (LTV_ERR_UNSUPPORTED past them): page_size <= 2^20, table_width * page_size
 * <= 2^31 - 1024, total < 2^31.
 * ---------------------------------------------------------------------- */
typedef struct ltv_paged_batch {
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* slots;
  const int32_t* starts;
  int64_t table_stride;
  int64_t total; /* rows of the token tensors: B * T without starts */
  int B, T, num_slots, num_pages, table_width, page_size;
} ltv_paged_batch;

/* Writes the new tokens' keys and values into their pages.
 * k, v: token rows (NKVH, D), strides (sequence, token, head); the sequence stride
 * is not used with starts.  Any alignment.  B <= 65,535, and total * NKVH * D < 2^31
 * elements where rows are not 16-byte aligned, else units of 16 bytes.  No reference
 * counterpart (its cache is contiguous: nanochat/kv_cache.py insert_kv). */
int ltv_paged_cache_append(int dtype, const void* k, const int64_t k_strides[3], const void* v,
                           const int64_t v_strides[3], void* k_pages,
                           const int64_t k_page_strides[3], void* v_pages,
                           const int64_t v_page_strides[3], const ltv_paged_batch* batch, int NKVH,
                           int D, void* stream);

/* ------------------------------------------------------------------------
 * Attention of the new tokens over the cache (which holds them already):
 *   out[i, t, h] = sum_j p_j v_j,  p = softmax over positions j <= pos(i, t) of
 *                  scale q[i, t, h] . k_j,  heads h of one group of NH / NKVH
 *                  sharing a k/v head
 *   lse[i, t, h] = log sum_j exp(scale q . k_j)       (lse may be NULL)
 * A token without any key to attend to gives 0 and -inf.  Values and keys at
 * positions that a token does not attend to never reach its output, whatever bit
 * patterns they hold.
 *
 * q: strides (sequence, token, head), last stride 1, any alignment.  out: strides
 * likewise, 16-byte aligned rows.  lse: one float per (row, head), contiguous.
 * scale > 0, log2(e) scale finite.  D a multiple of 8, at most 128.  max_len: the longest
 * sequence expected (a hint: it chooses how many workgroups there are and, past 10^11
 * operations, how bfloat16 probabilities are rounded, not which keys are read).  The pages of a layer
 * lie within 32 GiB, with strides that are not negative; total * NH < 2^30.
 * workspace: ltv_paged_attention_workspace_size bytes, 16-byte aligned.
 * ---------------------------------------------------------------------- */
size_t ltv_paged_attention_workspace_size(int dtype, const ltv_paged_batch* batch, int NH,
                                          int NKVH, int D, int max_len);

int ltv_paged_attention(int dtype, const void* q, const int64_t q_strides[3],
                        const void* k_pages, const int64_t k_page_strides[3],
                        const void* v_pages, const int64_t v_page_strides[3],
                        const ltv_paged_batch* batch, void* out, const int64_t out_strides[3],
                        float* lse, void* workspace, size_t workspace_bytes, int NH, int NKVH,
                        int D, int max_len, float scale, void* stream);

/* ------------------------------------------------------------------------
 * The pages of all layers, for the calls that move pages: `layers` pairs of a k
 * and a v page array whose pages are dense blocks of block_bytes bytes (a multiple
 * of 16, less than 2^31), page_bytes apart, the layers layer_bytes apart; 16-byte
 * aligned.  A call copies less than 2^31 pieces of 8 KiB.
 * ---------------------------------------------------------------------- */
typedef struct ltv_page_blocks {
  void* k;
  void* v;
  int64_t k_page_bytes, k_layer_bytes;
  int64_t v_page_bytes, v_layer_bytes;
  int64_t block_bytes;
  int layers, num_pages;
} ltv_page_blocks;

/* The cache's bookkeeping, in place (compact does not use seq_lens; fork, free and
 * compact not page_size, which must be positive all the same). */
typedef struct ltv_page_state {
  int32_t* page_table;
  int32_t* seq_lens;
  int32_t* ref_counts;
  int64_t table_stride;
  int num_slots, table_width, num_pages, page_size;
} ltv_page_state;

/* Makes room for counts[i] >= 0 more tokens in slot slots[i] (n entries, distinct
 * slots): seq_lens grows, and pages are taken, the lowest free ones in the order of
 * the entries.  Where a slot's last page is only partly filled and shared with
 * another slot, the new tokens may not go there: the slot gets a copy of that page
 * (first of its new pages) and lets go of the shared one; among slots of one call
 * that all hold the page and no other does, the last keeps it.
 * *status: 0; or, with nothing changed at all, how many pages are missing (at most
 * 2^31 - 1); or -1 for a slot or count out of range or a sequence that its table row cannot
 * hold.  Where it is not 0 the new tokens must not be appended: they would overwrite the last
 * ones of seq_lens (a batch whose slots are -1 then has no sequences).
 * workspace: ltv_paged_cache_reserve_workspace_size bytes, 16-byte aligned. */
size_t ltv_paged_cache_reserve_workspace_size(int n, int num_pages);
int ltv_paged_cache_reserve(const ltv_page_state* state, const ltv_page_blocks* blocks,
                            const int32_t* slots, const int32_t* counts, int n, int32_t* status,
                            void* workspace, size_t workspace_bytes, void* stream);

/* Slot dst[i] becomes a copy of slot src[i] that shares its pages (n entries): what
 * dst held is let go.  dst entries are distinct and none is a src entry, except that
 * src[i] == dst[i] does nothing. */
int ltv_paged_cache_fork(const ltv_page_state* state, const int32_t* src, const int32_t* dst,
                         int n, void* stream);

/* Empties n slots: their pages are let go, their table rows cleared to -1. */
int ltv_paged_cache_free(const ltv_page_state* state, const int32_t* slots, int n, void* stream);

/* Copies page src[i] to page dst[i] in every layer (n entries; an entry with an id
 * outside [0, P) or src[i] == dst[i] does nothing; no dst is another dst or a src). */
int ltv_paged_cache_copy(const ltv_page_blocks* blocks, const int32_t* src, const int32_t* dst,
                         int n, void* stream);

/* Moves the pages in use to the lowest ids: with L of them, those at ids >= L move,
 * in ascending order, into the free ids < L; table and counts follow.  *live: L.
 * workspace: ltv_paged_cache_compact_workspace_size bytes, 16-byte aligned. */
size_t ltv_paged_cache_compact_workspace_size(int num_pages);
int ltv_paged_cache_compact(const ltv_page_state* state, const ltv_page_blocks* blocks,
                            int32_t* live, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Log probabilities of given tokens, entropy and top alternatives, per row of
 * logits x (N, V), row stride row_stride, last stride 1:
 *   z = softcap tanh(x / softcap)   (softcap 0: z = x),  lse = log sum exp z
 *   logprobs[n]  = z[n, targets[n]] - lse;  0 for a target outside [0, V)
 *   entropy[n]   = -sum p log p,  p = exp(z - lse)      (may be NULL)
 *   top_ids[n, i], top_logprobs[n, i], 0 <= i < top_k <= 64, top_k <= V: the largest
 *                  logits in descending order of x (NaN above all), equal ones in
 *                  ascending order of index
 *   lse[n]       : kept for the backward                (may be NULL)
 * All outputs contiguous; sums in fp32.  workspace: ltv_token_logprobs_workspace_size
 * bytes (0 where a row is not cut into pieces), 16-byte aligned.  N < 2^31.  Replaces
 * what nanochat's sampling and scoring do with log_softmax, gather and topk on the logits.
 * ---------------------------------------------------------------------- */
size_t ltv_token_logprobs_workspace_size(int64_t N, int V, int top_k);
int ltv_token_logprobs_forward(int dtype, const void* logits, int64_t row_stride,
                               const int64_t* targets, float* logprobs, float* entropy,
                               float* lse, float* top_logprobs, int64_t* top_ids,
                               void* workspace, size_t workspace_bytes, int64_t N, int V,
                               int top_k, float softcap, void* stream);

/* Gradient of the above for the logits, (N, V) in their dtype:
 *   dz_j = g_logp (1[j = target] - p_j) - g_entropy p_j (log p_j + entropy)
 *          + sum_i g_top[i] (1[j = top_ids[i]] - p_j),   dx = dz (1 - (z / softcap)^2)
 * g_logprobs, g_entropy, g_top may be NULL (zero); entropy is read with g_entropy,
 * top_ids with g_top. */
int ltv_token_logprobs_backward(int dtype, const void* logits, int64_t row_stride,
                                const int64_t* targets, const float* lse, const float* entropy,
                                const int64_t* top_ids, const float* g_logprobs,
                                const float* g_entropy, const float* g_top, void* grad_logits,
                                int64_t grad_row_stride, int64_t N, int V, int top_k,
                                float softcap, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOCHAT_SERVING_AMD_H */
