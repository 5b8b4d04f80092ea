/*
 * jacq_kivi_attend.h -- C ABI of attention of chunks of queries over the int4
 * KIVI cache of libjacq_kivi.so (gfx950), and of its read-back.
 *
 * jacq_kivi.h writes the cache and decodes one query per sequence over all of
 * it; here are prompts and parts of prompts, several queries per sequence,
 * sliding windows with sinks, and queries that see every token (a decoder's
 * over the states of an encoder).  No counterpart in the reference.
 * Conventions, geometry, tensor layouts and the split into int4 groups and an
 * fp16 residual window are those of jacq_kivi.h; messages are in
 * jacq_kivi_last_error().
 *
 * Token t of a sequence of n tokens is int4 if it lies before
 *   old = max(0, n - R) / 32 * 32  (at most what the table addresses)
 * with K = code * scale + zero of its group and channel, V = code * scale +
 * zero of itself and its 32 channels; else it is row t - old of the scratch.
 * The products take both rounded to fp16 once, queries in fp16 (bf16 ones times
 * a power of two of the row) and softmax weights rounded to fp16; sums, maxima
 * and LSE are fp32.  An output of fp16 or fp32 is off by about 6e-4 of its norm,
 * mostly by K's rounding, where the codes hold K to a thirtieth of a group's
 * range.  A token that a query does not see may hold
 * anything.  To a query that sees it, a V that is not finite (fp16 V; or zero
 * or zero + 15 scale of 32 of its channels beyond fp16) counts as a NaN key:
 * all of the query's output is NaN.  A table entry outside
 * [0, num_pages) is never dereferenced: its tokens, and if it is a group's
 * first, which holds the scales of K, the group's, are NaN to the queries
 * that see them, and are read as NaN.  Lengths are clamped on the device to
 * [0, jacq_kivi_max_seq_len].
 */
#ifndef JACQ_KIVI_ATTEND_H
#define JACQ_KIVI_ATTEND_H

#include "jacq_kivi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of queries, outputs and read values */
#define JACQ_KIVI_FP16 0
#define JACQ_KIVI_BF16 1
#define JACQ_KIVI_FP32 2

/* The cache's arrays, as jacq_kivi_decode takes them. */
typedef struct jacq_kivi_pool {
  const uint8_t* k_code;
  const jacq_half_t* k_scale;
  const jacq_half_t* k_zero;
  const uint8_t* v_code;
  const jacq_half_t* v_scale;
  const jacq_half_t* v_zero;
  const jacq_half_t* k_scratch;
  const jacq_half_t* v_scratch;
} jacq_kivi_pool;

/* Sequence b has the queries CU_Q[b] to CU_Q[b + 1] of Q (one each when CU_Q
 * is NULL).
 *   causal 1  they are its last tokens: query i of m stands at position
 *             SEQ_LENS[b] - m + i and sees the tokens j <= position with
 *             j < sinks or j > position - window (all j <= position when
 *             window is 0)
 *   causal 0  every query sees all SEQ_LENS[b] tokens; no window
 * A query that sees nothing gives 0 (lse -inf), one whose scores all are -inf
 * NaN (lse -inf), as the definition's 0 / 0.  Scores are scale (> 0, finite
 * times log2(e)) times the products.
 *   Q    [total_q, NH, HD] of q_dtype (fp16 or bf16), token rows q_stride
 *        elements apart
 *   O    [total_q, NH, HD] of o_dtype (q_dtype or fp32), contiguous; may be Q
 *        where that has its type and stride
 *   LSE  NULL or [total_q, NH] fp32: log of the sum of exp(scaled scores)
 *   max_q  no sequence has more queries than this (of one that has, the first
 *        max_q are computed, at their own positions; the others are left alone)
 * Rows of Q and O outside every sequence's queries are not touched.  The
 * workspace needs no particular contents; calls that can run at the same time
 * must not share one.  No call synchronises, allocates or records a memset. */
typedef struct jacq_kivi_attend_args {
  const void* Q;
  const int32_t* CU_Q;
  const int32_t* SEQ_LENS;
  const int32_t* BLOCK_TABLES;
  void* O;
  float* LSE;
  int64_t q_stride;
  int32_t q_dtype, o_dtype;
  int32_t batch, total_q, max_q;
  int32_t window, sinks, causal;
  float scale;
} jacq_kivi_attend_args;

/* Depends on the current device's number of compute units. */
size_t jacq_kivi_attend_workspace_size(const jacq_kivi_geometry* geo, int32_t batch, int32_t total_q,
                                       int32_t max_q);
int jacq_kivi_attend(const jacq_kivi_geometry* geo, const jacq_kivi_pool* pool,
                     const jacq_kivi_attend_args* args, void* workspace, size_t workspace_bytes,
                     hipStream_t stream);

/* The values of tokens STARTS[b] to ENDS[b] of each sequence of ENDS[b] tokens,
 * one sequence after another: K, V [total, NKV, HD] of `dtype`, each rounded to
 * it once (bf16: from its fp32 value, which differs from the exact one only where
 * scale and zero are 2^9 apart or more).  Tokens past `total` are dropped. */
int jacq_kivi_read(const jacq_kivi_geometry* geo, const jacq_kivi_pool* pool, const int32_t* STARTS,
                   const int32_t* ENDS, const int32_t* BLOCK_TABLES, int32_t batch, int32_t total,
                   void* K, void* V, int32_t dtype, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* JACQ_KIVI_ATTEND_H */
