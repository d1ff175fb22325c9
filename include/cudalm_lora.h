/*
 * cudalm_lora -- C ABI of low-rank adapters of many requests beside shared
 * projections on the MI355X (gfx950). No counterpart in the reference.
 *
 * Every row m of the activations x[M][K] belongs to a request, and that to an adapter
 * index[m] or to none. Beside up to 8 projections of the same x (q/k/v, gate/up, or
 * one), whose results are y_j[M][N_j],
 *
 *   out_j[m] = y_j[m] + scales[i] * B_j[i] (A_j[i] x[m]),     i = index[m]
 *
 * with A_j [adapters][rank][K] and B_j [adapters][N_j][rank], row-major, in the type of
 * x and y (bf16 or fp16). A x is summed in fp32 and enters the second product as two
 * bf16 numbers (16 bits or more of it), fp16 factors as two each; sums and y are fp32,
 * the result is rounded once. Rows of no adapter keep y. Inf and NaN of a row, or of
 * an adapter that it does not have, reach no other row.
 *
 * Which rows have which adapter is laid out once per batch (cudalm_lora_plan), for
 * all projections of all layers of a step.
 *
 * Ownership, threading and errors are those of cudalm_w4a16.h: the caller owns every
 * buffer, calls keep no state, never synchronize and enqueue on `stream`; the same
 * CUDALM_W4A16_E* codes (EINVAL: a size or type that is not served; ENULL: a required
 * pointer is NULL; EALIGN: x, A, B or a plan that is not 16-byte aligned, or x's
 * row stride no multiple of 8, other bases below their elements' alignment; ERANGE: more
 * work than one launch or index holds, or a buffer that is too small). A plan may be
 * read by any number of calls at a time.
 */
#ifndef CUDALM_LORA_H
#define CUDALM_LORA_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "cudalm_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CUDALM_LORA_BF16 0
#define CUDALM_LORA_F16 1
#define CUDALM_LORA_MAX_PROJ 8
#define CUDALM_LORA_MAX_RANK 256
#define CUDALM_LORA_MAX_ADAPTERS 4096

typedef struct cudalm_lora_proj {
  const void* a; /* [adapters][rank][K] */
  const void* b; /* [adapters][N][rank] */
  const void* y; /* [M] rows of N, y_stride elements apart */
  void* out;     /* the same, out_stride apart; may be y, with its stride, and overlaps
                    nothing else of the call: not x, no other projection's y or out (EINVAL
                    where strides are the same, or M is 1; else the caller's part) */
  int64_t y_stride, out_stride;
  int N;
} cudalm_lora_proj;

/* Lays out index[M] (device, int32) for cudalm_lora_add: rows of one adapter together.
 * A number outside [0, adapters) means none. `plan` holds cudalm_lora_plan_bytes(M,
 * adapters) bytes (0: sizes that are not served), 16-byte aligned. */
size_t cudalm_lora_plan_bytes(int M, int adapters);
int cudalm_lora_plan(const int32_t* index, int M, int adapters, void* plan, size_t plan_bytes,
                     hipStream_t stream);

/* The sums above for `count` projections. K and rank are multiples of 8 (rank at
 * most 256). plan: made for the same M and adapters. scales: [adapters] fp32, device
 * (NULL: 1). ranks: [adapters] int32, device (NULL: `rank` each): how many rows of A and
 * columns of B adapter i uses; what stands in the others (padding) has no effect. */
int cudalm_lora_add(const cudalm_lora_proj* projs, int count, const void* x, int64_t x_stride, int K,
                    int M, int rank, int adapters, int type, const float* scales, const int32_t* ranks,
                    const void* plan, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
