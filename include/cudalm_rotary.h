/*
 * cudalm_rotary -- C ABI of rotary positions on the MI355X (gfx950): rows of heads
 * rotated by their positions, and new tokens' keys rotated on their way into the
 * pages of the paged cache (cudalm_paged_kv.h), with their queries.
 *
 * It serves the place of the reference's partial rotation
 * (src/kernels/qwen35_kernels.cu:40-479, batch twins batch_decode.cu:238-599), which
 * is one axis, channels i and pairs + i, and a pass of its own.
 *
 * A head of D channels has `pairs` pairs in its first 2 * pairs channels; pair i
 * is turned by the angle
 *
 *   w = p * freqs[i],    y0 = scale * (x0 cos w - x1 sin w)
 *                        y1 = scale * (x1 cos w + x0 sin w)
 *
 * and the channels behind are copied. p is the token's position on the pair's axis:
 * 1 to 4 axes (one for text; time, height and width for video) share the pairs out,
 * axis 0 .. axes - 1 getting sections[0 .. axes - 1] of them. Frequencies are taken
 * as exact numbers, angles made and reduced in 64-bit floats: w is off by less than
 * 2^-51 |w| (2^-27 at a position of 2^24 and a frequency of 1, 2^-20 at 2^31); the rest is
 * fp32, rounded once.
 *
 * Ownership, threading and errors are those of cudalm_w4a16.h: the caller owns every
 * buffer, calls keep no state, never synchronize and enqueue on `stream`; the same
 * CUDALM_W4A16_E* codes (EINVAL: a size, type or layout that is not served; ENULL: a
 * required pointer is NULL; EALIGN: a base below its elements' alignment or, in
 * append, a base or stride that is not 16-byte aligned; ERANGE: more work than one
 * launch holds).
 */
#ifndef CUDALM_ROTARY_H
#define CUDALM_ROTARY_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "cudalm_paged_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CUDALM_ROTARY_MAX_AXES 4
#define CUDALM_ROTARY_MAX_PAIRS 256

typedef struct cudalm_rotary {
  const float* freqs; /* [pairs], device: radians per position */
  int pairs;          /* 1 .. 256 */
  int adjacent;       /* 0: pair i is channels i and pairs + i; 1: 2 i and 2 i + 1 */
  int axes;           /* 1 .. 4 */
  int sections[CUDALM_ROTARY_MAX_AXES]; /* pairs of each axis, `pairs` in all */
  int turns;   /* 0: an axis' pairs lie together, axis 0's first; 1: pairs are dealt
                  to the axes in turn, an axis that has all of its own being passed over */
  float scale; /* of the rotated channels, normally 1 */
} cudalm_rotary;

/* Rows of heads with any strides (in elements; a head's D channels are contiguous). */
typedef struct cudalm_rotary_rows {
  const void* x;
  void* out; /* may be x itself, with x's strides: rotated in place; else it overlaps x nowhere,
                nor k or v of append. Its rows are apart. (EINVAL where rows of out share
                places, or, if strides are the same, with rows that are read) */
  int64_t x_token_stride, x_head_stride, out_token_stride, out_head_stride;
  int heads;
} cudalm_rotary_rows;

/* Rotates tokens x heads rows of head_dim channels (2 * pairs .. 512; type
 * CUDALM_PAGED_BF16 or _F16): row t by positions[axis * tokens + t] (device, int32, any
 * sign). Any alignment is served; 16-byte aligned bases, strides and head_dim that are
 * multiples of 8, and pairs that are, go 16 bytes at a time; the same of 8 bytes and
 * 4, 8 bytes at a time; others 2. */
int cudalm_rotary_rotate(const cudalm_rotary* rotary, const cudalm_rotary_rows* rows, int tokens,
                         int head_dim, int type, const int32_t* positions, hipStream_t stream);

/* cudalm_paged_append with rotated keys: rows cu_new[b] .. cu_new[b + 1] - 1 (NULL: tokens
 * / batch for every sequence) of k and v, [tokens][kv_heads][D], are the last tokens of
 * sequence b; keys are rotated and written into its pages, values written, weights set
 * to zero where kv->weights is not NULL. queries (NULL: none): those tokens' queries, rotated
 * by the same positions into queries->out; rows that belong to no sequence are not
 * written. Tokens of absent pages and before the first place are not cached, their
 * queries are rotated all the same. positions: [axes][tokens]; NULL: every axis of a
 * token is its place in the cache, lens[b] - n + j. (After an eviction a token's place
 * is not its position; the kept keys stay as they were rotated.) pairs is a multiple of
 * 8, at most D / 2; a query head count of any size; strides are multiples of 8. */
int cudalm_rotary_append(const cudalm_rotary* rotary, const cudalm_paged_kv* kv, const void* k,
                         const void* v, int64_t k_token_stride, int64_t k_head_stride,
                         int64_t v_token_stride, int64_t v_head_stride,
                         const cudalm_rotary_rows* queries, const int32_t* positions,
                         const int32_t* cu_new, int tokens, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
