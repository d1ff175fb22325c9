/*
 * cudalm_paged_kv -- C ABI of the MI355X (gfx950) paged key-value cache:
 * writing new tokens, attention over the pages for decode steps and prefill
 * chunks, and eviction by accumulated attention weight.
 *
 * It serves the place of the reference's paged cache and attention
 * (src/kernels/paged_kv.cu:53-180, batch twins batch_decode.cu:238-599) in
 * layouts of its own. One layer's cache is a pool of pages of P tokens:
 *
 *   k       : [num_pages][kv_heads][P][D]       16-bit, a token's key is a row
 *   v       : [num_pages][kv_heads][P/8][D][8]  16-bit, eight tokens interleaved:
 *             16 bytes hold one channel of eight tokens, which is what a matrix
 *             operand that sums over tokens wants from one load
 *   weights : [num_pages][kv_heads][P]          fp32, attention weight (optional)
 *
 * D (head_dim) is 64, 128 or 256, P a power of two of 16 .. 1024, the type
 * bf16 or fp16. tables[b][i] is the page of tokens [i P, (i + 1) P) of
 * sequence b; an entry outside [0, num_pages) means that these tokens are
 * absent (not allocated, or freed behind a sliding window): nothing reads or
 * writes them and no query sees them. lens[b] is the number of tokens of
 * sequence b, new ones included; it counts as at most max_pages * P, and as 0
 * where it is negative. Pages of different sequences may be shared as long as
 * no call writes them.
 *
 * Visibility. New token j of the n new ones of a sequence of L tokens has
 * position p = L - n + j and sees the cached tokens t with
 *
 *   0 <= t <= p   and   (window <= 0 or t > p - window or t < sinks)
 *
 * out = sum_t softmax_t(scale * q . k_t) v_t over the tokens it sees, and
 * zeros where it sees none (p < 0, absent pages) or where every score is
 * -inf. Inf and NaN in the values that it sees count whatever their weights,
 * also ones that underflow or are zero next to others. Whatever stands in places
 * that no query sees (NaN included) has no effect. Query head h reads key-value head h / (heads / kv_heads). Scores,
 * statistics and sums are fp32, and so is what kv->weights receives; a softmax weight
 * is rounded to the values' type before it meets them (the matrix unit takes no wider
 * ones), the sum that it is divided by is not; outputs are rounded once.
 *
 * Ownership, threading and errors are those of cudalm_w4a16.h: the caller
 * owns every buffer, calls keep no state, never synchronize and enqueue on
 * `stream`; the same CUDALM_W4A16_E* codes (EINVAL: a size, type or layout
 * that is not served; ENULL: a required pointer is NULL; EALIGN: a base or
 * stride that is not 16-byte aligned (fp32 and int32 bases: 4); ERANGE: more
 * work than one launch or index holds, or a workspace that is too small).
 * A workspace serves one call at a time, on any stream.
 */
#ifndef CUDALM_PAGED_KV_H
#define CUDALM_PAGED_KV_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "cudalm_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CUDALM_PAGED_BF16 0
#define CUDALM_PAGED_F16 1

/* A layer's cache and the sequences of a call. */
typedef struct cudalm_paged_kv {
  void* k;
  void* v;
  float* weights;        /* may be NULL where a call does not use them */
  const int32_t* tables; /* [batch][max_pages], device */
  const int32_t* lens;   /* [batch], device */
  int num_pages, page_size, kv_heads, head_dim, type;
  int batch, max_pages;
} cudalm_paged_kv;

/* Queries and options of an attention call. Strides are in elements,
 * multiples of 8; a head's D elements are contiguous. out is contiguous
 * [rows][heads][D]. */
typedef struct cudalm_paged_query {
  const void* q;
  void* out;
  int64_t token_stride, head_stride;
  int heads;   /* query heads, a multiple of kv_heads, at most 64 per kv head */
  float scale; /* of the scores, normally D^-1/2 */
  int window;  /* <= 0: none */
  int sinks;   /* first tokens that stay visible behind the window */
  int max_len; /* no sequence is expected to be longer (<= 0: max_pages *
                  page_size): the split of the work goes by it, and decode's
                  room for weights, which are zero past it */
} cudalm_paged_query;

/* Writes the keys and values of the new tokens of every sequence into its
 * pages, and zeros into their weights where kv->weights is not NULL. Rows
 * cu_new[b] .. cu_new[b + 1] - 1 (device, [batch + 1]) of k and v, [tokens]
 * [kv_heads][D] with the given strides, are the last tokens of sequence b;
 * cu_new NULL: every sequence has tokens / batch new ones. */
int cudalm_paged_append(const cudalm_paged_kv* kv, const void* k, const void* v,
                        int64_t k_token_stride, int64_t k_head_stride,
                        int64_t v_token_stride, int64_t v_head_stride,
                        const int32_t* cu_new, int tokens, hipStream_t stream);

/* Attention of the last `new_tokens` tokens of every sequence (rows
 * b * new_tokens + j of q and out); their keys and values are in the cache.
 * new_tokens * heads / kv_heads is at most 1024.
 * weights_mode: 0 none; CUDALM_PAGED_WEIGHTS_SET / _ADD: the weight of every
 * token t < lens[b], summed over the new tokens and the query heads of its
 * key-value head, replaces / is added to kv->weights (zero for tokens that no
 * query sees). That counts every new token of the call: with drafted tokens,
 * also those that are refused afterwards (to leave them out, decode the accepted
 * ones alone with weights, after verification). A page that two sequences of the
 * call share gets the weights of one of them, unspecified which. */
#define CUDALM_PAGED_WEIGHTS_SET 1
#define CUDALM_PAGED_WEIGHTS_ADD 2
size_t cudalm_paged_decode_workspace_bytes(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                                           int new_tokens, int weights_mode);
int cudalm_paged_decode(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int new_tokens,
                        int weights_mode, void* workspace, size_t workspace_bytes,
                        hipStream_t stream);

/* The same, without weights, where groups of sequences begin with the same tokens, whose
 * pages are read once for all of a group's queries. Group g is sequences cu[g] .. cu[g + 1] - 1
 * (device, [count + 1], ascending within 0 .. batch; sequences of no group share
 * nothing); its first shared[g] tokens (device, [count]; any number, below zero counts as
 * zero) are those in the pages of its first sequence, past its length too, and what the other
 * sequences' tables hold for them does not count (of a page that is shared in part they hold the
 * rest). A sequence need not have them all: it sees those of its length. Where every
 * table names the same pages, results are those of cudalm_paged_decode but for rounding.
 * (Bounds that do not ascend make their sequences' results unspecified; nothing outside of the
 * tensors is touched.) Every sequence's row of out is written. */
typedef struct cudalm_paged_groups {
  const int32_t* cu;
  const int32_t* shared;
  int count;      /* 1 .. batch */
  int max_shared; /* no group is expected to share more (<= 0: max_pages * page_size); only
                     speed goes by it */
} cudalm_paged_groups;
size_t cudalm_paged_decode_shared_workspace_bytes(const cudalm_paged_kv* kv,
                                                  const cudalm_paged_query* q,
                                                  const cudalm_paged_groups* groups, int new_tokens);
int cudalm_paged_decode_shared(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                               const cudalm_paged_groups* groups, int new_tokens, void* workspace,
                               size_t workspace_bytes, hipStream_t stream);

/* Attention of a chunk: rows cu_new[b] .. cu_new[b + 1] - 1 (device,
 * [batch + 1], ascending from 0 to `tokens`) of q and out are the last tokens
 * of sequence b; their keys and values are in the cache. Rows that belong to no
 * sequence are not written. (Ranges that do not ascend or leave 0 .. tokens make
 * their rows' results unspecified; nothing outside of the tensors is touched.) */
size_t cudalm_paged_prefill_workspace_bytes(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                                            int tokens);
int cudalm_paged_prefill(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                         const int32_t* cu_new, int tokens, void* workspace,
                         size_t workspace_bytes, hipStream_t stream);

/* Eviction. Of the present tokens of every sequence and key-value head it
 * keeps `keep` (all, where there are no more): the first min(sinks, keep)
 * positions, the last min(recent, keep - sinks) ones and, of the others, those
 * with the largest kv->weights (NaN counts as less than any number; equal
 * weights: the earlier token). The kept tokens' keys, values and weights are
 * copied, in their order, into the pages of dst_tables [batch][dst_pages],
 * and their old positions written to kept [batch][kv_heads][keep] (-1 past
 * the last); new_lens[b] is their number, and may be kv->lens itself. Other
 * places of the pages stay as they are. No page of dst_tables may be read
 * through kv->tables by the same call; dst_pages * P >= keep. Entries of
 * dst_tables outside [0, num_pages) drop the tokens that belong there from the
 * copy. max_len: no sequence is expected to be longer (<= 0: max_pages *
 * page_size); only speed goes by it. Every head keeps tokens of its own, so a
 * place of the new cache stands for another old position in each; positions,
 * windows and sinks of later calls count places. */
size_t cudalm_paged_evict_workspace_bytes(const cudalm_paged_kv* kv, int max_len);
int cudalm_paged_evict(const cudalm_paged_kv* kv, const int32_t* dst_tables, int dst_pages,
                       int keep, int sinks, int recent, int32_t* kept, int32_t* new_lens,
                       int max_len, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Registers of the attention kernels for a head_dim (VGPR + AGPR), -1 if
 * there is none: decode (prefill = 0) or prefill (1). */
int cudalm_paged_kernel_regs(int type, int head_dim, int prefill);

#ifdef __cplusplus
}
#endif

#endif
