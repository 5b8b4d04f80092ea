// q8_common.h -- shared definitions of the 8-bit paged cache's kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attend_common.h"
#include "jacq_q8.h"

namespace jacq {

static_assert(kFp16 == JACQ_Q8_FP16 && kBf16 == JACQ_Q8_BF16 && kFp32 == JACQ_Q8_FP32, "types");

namespace q8 {

constexpr float kFloor = 0x1p-24f;   // a block's largest magnitude counts as at least this
// Workgroups of the decode kernel that a CU holds (a wavefront of each a SIMD), by what its
// registers allow.
constexpr int decode_groups(int hd, int nb) { return (hd == 128 ? 4 : 5) - nb; }

struct Geo {
  int nh, nkv, hd, page, page_log2, max_pages, num_pages, gqa, codes;
};

struct Pool {
  const uint8_t* k_code;
  const float* k_scale;
  const uint8_t* v_code;
  const float* v_scale;
  const uint16_t* k_tail;
  const uint16_t* v_tail;
};

struct AppendArgs {
  jacq_q8_pool pool;
  const uint16_t* new_k;
  const uint16_t* new_v;
  int64_t k_stride, v_stride;
  const int32_t* cu;      // null: one token per sequence
  const int32_t* start;
  const int32_t* tables;
  int total, max_new, bf16;
};

struct AttendArgs {
  Pool pool;
  const uint16_t* q;
  const int32_t* cu;      // null: one query per sequence
  const int32_t* lens;
  const int32_t* tables;
  void* o;
  float* lse;             // null: not wanted
  float* weights;
  int64_t q_stride;
  int q_bf16, o_type;     // o_type: JACQ_Q8_*
  int batch, total_q, max_q;
  int window, sinks;      // window 0: none
  float scale;            // log2(e) included
  float decay;
  // split pieces and the sums of 16-token groups
  float* part_ml;         // decode: [target + segments][rows][2]; prefill: [slices][total_q][nh][2]
  float* part_acc;        // the same [HD]
  float* group_lse;       // [batch][nkv][row blocks][groups][rows]
  float* row_lse;         // [total_q][nh], base 2
  int32_t* plan;          // decode of many sequences: [batch + 1] first slices, then their size
  int target;             // decode: slices to aim at; 0: segments stay whole
  int cus;                // compute units
  int rows;               // rows of a segment at most (<= 16 NB)
  int row_blocks;         // row blocks of a sequence at most
  int groups;             // 16-token groups a table addresses
  int slices;             // prefill: workgroups that share a row tile's tokens, at most
  float load;             // row tiles a CU
  unsigned tiles, merges; // prefill: its units of row tiles, and its merge's (Place)
};

// Four codes (one dword) as fp16, exactly: what the matrix cores take.
//  int8: the byte u = code + 128 under the exponent of 1024 is 1024 + u; minus 1152 is the code.
//  e4m3: the conversion instruction with scale 1.
template <bool E4M3>
__device__ inline void codes4(uint32_t w, h2& lo, h2& hi) {
  if constexpr (E4M3) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true);
  } else {
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
  }
}

template <bool E4M3>
__device__ inline h8 codes8(uint32_t w0, uint32_t w1) {
  h2 a, b, c, d;
  codes4<E4M3>(w0, a, b);
  codes4<E4M3>(w1, c, d);
  h8 r;
  r.s01 = a;
  r.s23 = b;
  r.s45 = c;
  r.s67 = d;
  return r;
}

__device__ inline int clamp_len(const Geo& g, int n) {
  const int cap = g.max_pages << g.page_log2;  // the host checked that this fits
  return n < 0 ? 0 : n > cap ? cap : n;
}

// The tiles of kTile tokens that the queries of a sequence of n tokens may see, in order: the
// sinks' tiles, the window's, then the tail (fp16) as a unit of its own.
struct Span {
  int n;        // tokens
  int first;    // the lowest position of a query (may be negative)
  int nq;       // of them quantised
  int w0;       // first tile of the window
  int ns;       // tiles of the sinks before it
  int tiles;    // quantised tiles in all
  int units;    // units of a segment, at least 1 (a segment without tokens still writes its zeros)
  __device__ Span() {}
  __device__ Span(const Geo& g, int n_, int first_, int window, int sinks) {
    n = n_;
    first = first_;
    nq = n >> g.page_log2 << g.page_log2;
    tiles = (nq + kTile - 1) / kTile;
    w0 = ns = 0;
    if (window > 0 && first >= window) {
      w0 = (first - window + 1) / kTile;
      w0 = w0 > tiles ? tiles : w0;
      const int s = sinks < n ? sinks : n;
      ns = (int)(((int64_t)s + kTile - 1) / kTile);
      ns = ns > w0 ? w0 : ns;
    }
    units = ns + tiles - w0 + (n > nq ? 1 : 0);
    units = units < 1 ? 1 : units;
  }
  __device__ int tile_of(int u) const { return u < ns ? u : w0 + u - ns; }  // == tiles: the tail
};

inline __device__ Span make_span(const Geo& g, const AttendArgs& a, int n, int all) {
  return Span(g, n, n - all, a.window, a.sinks);
}

__device__ inline int row_slices(const Geo&, const AttendArgs& a, const Place& p) {
  return prefill_slices(a, p.n);
}

hipError_t launch_append(const Geo& g, const AppendArgs& a, int batch, hipStream_t s);
hipError_t launch_read(const Geo& g, const Pool& p, const int32_t* starts, const int32_t* ends,
                       const int32_t* tables, int batch, int total, void* k, void* v, int type,
                       hipStream_t s);
hipError_t launch_decode(const Geo& g, const AttendArgs& a, int nb, hipStream_t s);
hipError_t launch_decay(const Geo& g, const AttendArgs& a, hipStream_t s);  // of a call of no queries
hipError_t launch_prefill(const Geo& g, const AttendArgs& a, hipStream_t s);
hipError_t launch_evict(const Geo& g, const float* w, const int32_t* lens, const int32_t* tables,
                        int batch, int keep, int sink, int recent, int32_t* tables_out,
                        int32_t* lens_out, float* w_out, int32_t* evicted, hipStream_t s);

}  // namespace q8

template <>
struct SpanOf<q8::Geo> {
  typedef q8::Span type;
};

}  // namespace jacq
