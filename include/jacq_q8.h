/*
 * jacq_q8.h -- C ABI of the 8-bit paged KV cache of libjacq_kivi.so (gfx950).
 *
 * The int4 KIVI cache (jacq_kivi.h) holds 4 bits per value and an fp16 window;
 * this one holds 8 bits per value with one scale per block of tokens and kv
 * head, and nothing in fp16 but the block in progress.  It has no counterpart
 * in the reference.  Conventions are those of jacq_kivi.h: caller-owned device
 * memory, calls asynchronous on `stream` (a stream of the current device),
 * status codes (JACQ_KIVI_*) with the message in jacq_q8_last_error().
 *
 * A block is a page of P tokens (16, 32 or 64).  For one kv head of a block,
 * with A = max(|x|, 2^-24) over its P x HD values x:
 *   int8   scale = A / 127, code = round_half_even(127 x / A), stored + 128
 *   e4m3   scale = A / 448, code = 448 x / A rounded half to even to e4m3
 * and the value is code * scale.  A block is quantised when its last token
 * arrives, from all its tokens, so its bits do not depend on how they came.
 * Until then its tokens stay fp16 in the sequence's tail.  Values enter as
 * fp16: bf16 values of magnitude 2^-14 to 65504 exactly, smaller ones to
 * within 2^-25, larger ones and infinities as +-65504.  A NaN in a token's K
 * or V makes the token's key NaN in that kv head (its V is stored as 0), and
 * the scale of K NaN when the block is quantised: every query that sees the
 * token, or the block once quantised, gives NaN; no other query does.
 *
 * Tensor layouts (row-major):
 *   K_CODE        uint8  [num_pages, NKV, P, HD]
 *   V_CODE        uint8  [num_pages, NKV, HD, P]   (a channel's tokens side by side)
 *   K/V_SCALE     fp32   [num_pages, NKV]
 *   K/V_TAIL      fp16   [batch, NKV, P, HD]: tokens len / P * P ... len - 1
 *   BLOCK_TABLES  int32  [batch, max_pages_per_seq]
 *   weights       fp32   [batch, max_pages_per_seq]
 * Lengths are clamped on the device to [0, max_pages_per_seq * P]; of a
 * sequence whose length before an append is outside [0, that) all new tokens
 * are dropped.  A table
 * entry outside [0, num_pages) is never dereferenced: a read of it gives NaN,
 * a write to it is dropped.
 */
#ifndef JACQ_Q8_H
#define JACQ_Q8_H

#include "jacq_kivi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JACQ_Q8_VERSION 1

/* code types */
#define JACQ_Q8_INT8 0
#define JACQ_Q8_E4M3 1
/* element types of queries, new tokens and outputs */
#define JACQ_Q8_FP16 0
#define JACQ_Q8_BF16 1
#define JACQ_Q8_FP32 2

/* The most queries per sequence of a call that adds up block weights. */
#define JACQ_Q8_MAX_WEIGHTED_QUERIES 64
/* The widest block table. */
#define JACQ_Q8_MAX_PAGES_PER_SEQ 16384

typedef struct jacq_q8_geometry {
  int32_t num_heads;         /* NH */
  int32_t num_kv_heads;      /* NKV; NH % NKV == 0, NH / NKV <= 16 */
  int32_t head_dim;          /* HD: 64 or 128 */
  int32_t page_size;         /* P: 16, 32 or 64 */
  int32_t max_pages_per_seq; /* block-table row width, 1 to 16384 */
  int32_t num_pages;         /* physical pages in the pool */
  int32_t codes;             /* JACQ_Q8_INT8 or JACQ_Q8_E4M3 */
} jacq_q8_geometry;

typedef struct jacq_q8_pool {
  uint8_t* k_code;
  float* k_scale;
  uint8_t* v_code;
  float* v_scale;
  jacq_half_t* k_tail;
  jacq_half_t* v_tail;
} jacq_q8_pool;

int jacq_q8_version(void);
const char* jacq_q8_last_error(void);
int jacq_q8_check_geometry(const jacq_q8_geometry* geo);
int64_t jacq_q8_max_seq_len(const jacq_q8_geometry* geo);

/* Append new tokens to each of `batch` sequences.
 *   NEW_K/NEW_V  [total_new, NKV, HD] fp16 or bf16 (`dtype`), a token's row
 *                k_stride / v_stride elements after the one before
 *   CU_NEW       [batch + 1] int32: sequence b's tokens are rows CU_NEW[b] to
 *                CU_NEW[b + 1]; NULL: one token per sequence (total_new = batch)
 *   START_LENS   [batch] int32, lengths before the append
 *   max_new      no sequence has more new tokens than this (more are dropped,
 *                as are tokens past the table's capacity) */
int jacq_q8_append(const jacq_q8_geometry* geo, const jacq_q8_pool* pool, const void* NEW_K,
                   const void* NEW_V, int32_t dtype, int64_t k_stride, int64_t v_stride,
                   const int32_t* CU_NEW, const int32_t* START_LENS,
                   const int32_t* BLOCK_TABLES, int32_t total_new, int32_t max_new,
                   int32_t batch, hipStream_t stream);

/* Attention of a call's queries over the cache.  Sequence b has the queries
 * CU_Q[b] to CU_Q[b + 1] of Q (one each when CU_Q is NULL), its last tokens:
 * query i of m stands at position SEQ_LENS[b] - m + i and sees the tokens
 * j <= position with j < sinks or j > position - window (all j <= position
 * when window is 0).  A query that sees nothing gives 0 (lse -inf).  Scores
 * are scale (> 0) times the products.
 *   Q        [total_q, NH, HD] of q_dtype, token rows q_stride elements apart
 *   O        [total_q, NH, HD] of o_dtype (q_dtype or fp32), contiguous
 *   LSE      NULL or [total_q, NH] fp32: log of the sum of exp(scaled scores)
 *   WEIGHTS  NULL or [batch, max_pages_per_seq] fp32: of every block, decay
 *            times what it held (decay 0 overwrites) plus the softmax weight
 *            of its tokens summed over the sequence's queries and heads;
 *            at most JACQ_Q8_MAX_WEIGHTED_QUERIES queries per sequence.  The
 *            workspace then holds a float for every row (query x head) of
 *            every 16 tokens that the table addresses, the rows of a kv head
 *            in 16s or 32s: batch x NKV x max_pages_per_seq x P / 4 x rows
 *            bytes, whatever the lengths are
 *   max_q    no sequence has more queries than this (of one that has, the
 *            first max_q are computed, at their own positions; the others are
 *            left alone)
 * Rows of Q and O outside every sequence's queries are not touched.  The
 * workspace needs no particular contents; calls that can run at the same time
 * must not share one. */
typedef struct jacq_q8_attend_args {
  const void* Q;
  const int32_t* CU_Q;
  const int32_t* SEQ_LENS;
  const int32_t* BLOCK_TABLES;
  void* O;
  float* LSE;
  float* WEIGHTS;
  int64_t q_stride;
  int32_t q_dtype, o_dtype;
  int32_t batch, total_q, max_q;
  int32_t window, sinks;
  float scale;
  float decay;
} jacq_q8_attend_args;

size_t jacq_q8_attend_workspace_size(const jacq_q8_geometry* geo, int32_t batch, int32_t total_q,
                                     int32_t max_q, int32_t weighted);
int jacq_q8_attend(const jacq_q8_geometry* geo, const jacq_q8_pool* pool,
                   const jacq_q8_attend_args* args, void* workspace, size_t workspace_bytes,
                   hipStream_t stream);

/* The values of tokens STARTS[b] to ENDS[b] of each sequence of ENDS[b] tokens
 * (the tail holds those from ENDS[b] / P * P on), one sequence after another:
 * K, V [total, NKV, HD] of `dtype`.  Tokens past `total` are dropped. */
int jacq_q8_read(const jacq_q8_geometry* geo, const jacq_q8_pool* pool, const int32_t* STARTS,
                 const int32_t* ENDS, const int32_t* BLOCK_TABLES, int32_t batch, int32_t total,
                 void* K, void* V, int32_t dtype, hipStream_t stream);

/* Evict the lightest blocks of every sequence with more than `keep` full
 * blocks: the first sink_pages and the last recent_pages full blocks stay, of
 * the others the heaviest until `keep` stay (of equal weights the earlier; NaN
 * is lightest).  sink_pages + recent_pages <= keep.  The kept entries of a
 * table row move to its front in order, the evicted ones follow in order (they
 * are the sequence's own spare pages), the rest of the row stays; the weights
 * move along, 0 behind them except the block in progress; the length drops by
 * P per evicted block.  No page moves.  Each OUT may be its input's buffer.
 *   EVICTED  [batch] int32, blocks evicted */
int jacq_q8_evict(const jacq_q8_geometry* geo, const float* WEIGHTS, const int32_t* SEQ_LENS,
                  const int32_t* BLOCK_TABLES, int32_t batch, int32_t keep, int32_t sink_pages,
                  int32_t recent_pages, int32_t* TABLES_OUT, int32_t* LENS_OUT,
                  float* WEIGHTS_OUT, int32_t* EVICTED, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* JACQ_Q8_H */
