/*
 * jacq_rotary.h -- C ABI of the rotary positions of queries and keys of
 * libjacq_kivi.so (gfx950): what new tokens go through before they are appended
 * to a cache and attend over it.  No counterpart in the reference.  Conventions
 * are those of jacq_kivi.h: caller-owned device memory, calls asynchronous on
 * `stream` (a stream of the current device), status codes JACQ_KIVI_* with the
 * message in jacq_rotary_last_error().
 *
 * Of a head's first rotary_dim channels, pair i (i < rotary_dim / 2) is the
 * channels i and i + rotary_dim / 2 (JACQ_ROTARY_HALF) or 2 i and 2 i + 1
 * (JACQ_ROTARY_INTERLEAVED).  A token at position p turns its pair (a, b) by the
 * angle t = p f_i:
 *   a' = amplitude (a cos t - b sin t),  b' = amplitude (b cos t + a sin t)
 * The other channels stay as they are.  f_i comes as the fraction of a turn of
 * one position, in 2^-64 of a turn (TURNS, host memory, read during the call):
 * the product with the position modulo 2^64 is the angle's fraction of a turn
 * exactly, whatever the position.  cos and sin are within 2^-22 of their values;
 * the rest is fp32, each output rounded to its type once.
 */
#ifndef JACQ_ROTARY_H
#define JACQ_ROTARY_H

#include "jacq_kivi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JACQ_ROTARY_HALF 0
#define JACQ_ROTARY_INTERLEAVED 1
/* element types */
#define JACQ_ROTARY_FP16 0
#define JACQ_ROTARY_BF16 1
#define JACQ_ROTARY_FP32 2
/* most channels of a head that turn */
#define JACQ_ROTARY_MAX_DIM 256

/*   Q, K        [tokens, heads, head_dim] of `dtype`, token rows q_stride and
 *               k_stride elements apart; K and K_OUT NULL with num_kv_heads 0
 *   Q_OUT, K_OUT  the same of q_out_dtype, k_out_dtype; each may be its input
 *               itself (same type and stride), else must not overlap any input
 *   POSITIONS   [tokens] int32, or int64 with positions64; any sign
 *   inverse     1: by the negative angles (with amplitude 1 the way back; with
 *               any, the gradient of the rotation for the gradient of its output) */
typedef struct jacq_rotary_args {
  const void* Q;
  const void* K;
  const void* POSITIONS;
  void* Q_OUT;
  void* K_OUT;
  const uint64_t* TURNS; /* host, [rotary_dim / 2] */
  int64_t q_stride, k_stride, q_out_stride, k_out_stride;
  int32_t tokens, num_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t layout, dtype, q_out_dtype, k_out_dtype, positions64, inverse;
  float amplitude;
} jacq_rotary_args;

const char* jacq_rotary_last_error(void);
int jacq_rotary(const jacq_rotary_args* args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* JACQ_ROTARY_H */
