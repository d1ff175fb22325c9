/*
 * cudalm_draft -- C ABI of the verification of drafted tokens: which of the
 * tokens that a draft model proposed the target model accepts, and the token
 * that follows them, so that the output is distributed as the target's.
 * The reference decodes one token per step and has no counterpart.
 *
 * target [batch][draft + 1][vocab]: the target's probabilities at the
 * position of every drafted token and after the last. draft_probs
 * [batch][draft][vocab]: the draft's, or NULL where it proposed its tokens
 * with certainty (probability 1 each). Both of the same type; values are
 * used as fp32. tokens [batch][draft] the drafted tokens, counts [batch] how
 * many of them there are (NULL: draft; clamped to 0 .. draft). u_accept
 * [batch][draft] and u_next [batch] are random numbers of [0, 1), fp32.
 *
 * Token x_i is accepted, in order, while
 *
 *   u_accept[i] * q_i(x_i) < p_i(x_i)            (fp32, one rounding)
 *
 * (a token outside the vocabulary, or a NaN, is not). With n accepted the
 * next token is drawn from max(p_n - q_n, 0) where one was refused, and from
 * p_n where none was, or where that difference is zero everywhere. The
 * draw inverts the cumulative sum of the probabilities in whole units of
 * 2^-40 (each clamped to [0, 1] and truncated), so it does not depend on an
 * order of summation: the token is the first v with
 *
 *   sum_{w <= v} r_w > floor(sum_w r_w * U / 2^24),   U = floor(u_next * 2^24)
 *
 * out [batch][draft + 1] gets the accepted tokens, the next one, and -1 in the
 * remaining places; accepted [batch] gets n, and may be counts itself. Where
 * p_n is zero everywhere the next token is -1.
 */
#ifndef CUDALM_DRAFT_H
#define CUDALM_DRAFT_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "cudalm_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CUDALM_DRAFT_F32 0
#define CUDALM_DRAFT_BF16 1
#define CUDALM_DRAFT_F16 2

/* Row strides in elements (of consecutive positions; sequences are
 * draft + 1 and draft rows apart). 1 <= vocab <= 2^22, draft >= 0. */
size_t cudalm_draft_verify_workspace_bytes(int batch, int draft, int vocab);
int cudalm_draft_verify(const void* target, int64_t target_stride, const void* draft_probs,
                        int64_t draft_stride, int type, const int32_t* tokens,
                        const int32_t* counts, const float* u_accept, const float* u_next,
                        int32_t* out, int32_t* accepted, int batch, int draft, int vocab,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
