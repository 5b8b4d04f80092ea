// q8_common.h -- shared definitions of the 8-bit paged cache's kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jacq_q8.h"

namespace jacq {
namespace q8 {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kFloor = 0x1p-24f;   // a block's largest magnitude counts as at least this
constexpr int kTile = 64;            // tokens per step of the attention kernels
constexpr int kRowsLog2 = 7;
constexpr int kPrefillRows = 1 << kRowsLog2;  // query rows of a workgroup of the prefill kernel
constexpr int kSliceUnits = 8;       // tiles of one of its slices, about, at least (prefill_slices)
constexpr int kMaxSlices = 32;       // of its slices at most
// Workgroups of the decode kernel that a CU holds (a wavefront of each a SIMD), by what its
// registers allow.
constexpr int decode_groups(int hd, int nb) { return (hd == 128 ? 4 : 5) - nb; }
constexpr float kLog2e = 1.4426950408889634f;
// The weights 2^(t - m) that are rounded to fp16, the type that the matrix cores take at full rate
// with the most bits: m moves to kLift below a row's largest t, and only where that has passed m by
// kSlack more.  So they end at 2^15, the largest so far is at least 2^7, and the others keep 11 bits
// (half a step: 2^-11 of them) down to 2^-14, and are off by at most 2^-25 below.  O loses at most n
// 2^-32 of the largest |v| in the heaviest's block to that; the sum that divides it is of the
// unrounded weights, in fp32.
constexpr float kLift = 7.0f;
constexpr float kSlack = 8.0f;

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

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float log2_(float x) { return __builtin_amdgcn_logf(x); }
__device__ inline uint16_t f2bf(float f) {  // round to nearest even; NaN stays NaN
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}
// by value: a bit_cast of a vector's element in place takes the vector's first
__device__ inline uint16_t h_bits(_Float16 x) { return __builtin_bit_cast(uint16_t, x); }
__device__ inline uint16_t f2h_(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
__device__ inline float h2f_(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }

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

// Inclusive prefix over the 64 lanes, by DPP: shifts within rows of 16 lanes, then the last lanes of
// rows (0 is the identity of both operations on what is summed here).
template <class Op>
__device__ inline int wave_prefix(int x, Op op) {
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr:1
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return x;
}
struct Sum {
  __device__ int operator()(int a, int b) const { return a + b; }
};
struct SumF {  // of fp32 bits
  __device__ int operator()(int a, int b) const {
#pragma clang fp contract(off)
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  }
};
struct Max {  // of numbers that are not negative
  __device__ int operator()(int a, int b) const { return a > b ? a : b; }
};
__device__ inline int lane63(int x) { return __builtin_amdgcn_readlane(x, 63); }

__device__ inline int clamp_len(const Geo& g, int n) {
  const int cap = g.max_pages << g.page_log2;  // the host checked that this fits
  return n < 0 ? 0 : n > cap ? cap : n;
}

// Queries of sequence b: rows [q0, q0 + m) of Q, whatever the table of offsets holds.  m is at most
// max_q; `all` are the sequence's own, which its last tokens are.
__device__ inline void queries_of(const AttendArgs& a, int b, int* q0, int* m, int* all) {
  if (!a.cu) {
    *q0 = b;
    *m = *all = 1;
    return;
  }
  int lo = a.cu[b], hi = a.cu[b + 1];
  lo = lo < 0 ? 0 : lo > a.total_q ? a.total_q : lo;
  hi = hi < lo ? lo : hi > a.total_q ? a.total_q : hi;
  *q0 = lo;
  *all = hi - lo;
  *m = hi - lo > a.max_q ? a.max_q : hi - lo;
}

// Where a prefill's workgroup, or one of its merge, works.  A unit is 2^log2 rows of a sequence, `per`
// a query; the sequences' units follow each other, so a call's go by its queries and not by its
// sequences times max_q.  A unit of no rows is little work, but such units between the others leave
// those to few of a chiplet's engines (300 sequences of 1000 tokens with a query each, 40/8 heads of
// 128, under max_q 26 and 100, so with 1 and 3 empty ones each: 361 and 697 us, 217 and 237 without).
// Over the lanes of a wavefront alike, a sequence each.  Up to 64 sequences every one's units are
// counted; of more, one's units begin at (cu[b] per >> log2) + b, which leaves it as many as its rows
// begin or one more, and its sequence is found in every 64th offset first.
constexpr int kCounted = 64;
struct Place {
  int b, q0, m, all;  // sequence, and queries_of it
  int n;              // its tokens
  int at;             // which of its units; below 0: none
};
__device__ inline Place place_of(const Geo& g, const AttendArgs& a, int unit, int per, int log2) {
  const int lane = threadIdx.x & 63;
  auto offset = [&](int b) {
    const int x = a.cu[b];
    return x < 0 ? 0 : x > a.total_q ? a.total_q : x;
  };
  auto first = [&](int b, int q) { return ((int64_t)q * per >> log2) + b; };
  int at = 0, n = a.batch;
  while (n > 64) {
    const int step = (n + 63) / 64, i = lane * step;
    const int past = __popcll(__ballot(i < n && first(at + i, offset(at + (i < n ? i : 0))) <= unit));
    const int skip = past > 0 ? (past - 1) * step : 0;
    at += skip;
    n = step < n - skip ? step : n - skip;
  }
  const int b = at + (lane < n ? lane : n - 1), lo = offset(b), len = clamp_len(g, a.lens[b]);
  int hi = offset(b + 1);
  hi = hi < lo ? lo : hi;
  const int m = hi - lo > a.max_q ? a.max_q : hi - lo;
  int begin;
  uint64_t here;  // the last lane of these has the unit
  if (a.batch <= kCounted) {
    const int units = lane < n ? (int)(((int64_t)m * per + (1 << log2) - 1) >> log2) : 0;
    begin = wave_prefix(units, Sum()) - units;
    here = __ballot(unit >= begin && unit - begin < units);
  } else {
    begin = (int)first(b, lo);
    here = __ballot(lane < n && begin <= unit);
  }
  const int l = here ? 63 - __builtin_clzll(here) : 0;
  Place p;
  p.b = uniform(at + l);
  p.q0 = __builtin_amdgcn_readlane(lo, l);
  p.all = __builtin_amdgcn_readlane(hi, l) - p.q0;
  p.m = __builtin_amdgcn_readlane(m, l);
  p.n = __builtin_amdgcn_readlane(len, l);
  p.at = here ? unit - __builtin_amdgcn_readlane(begin, l) : -1;
  return p;
}

// Workgroups that share the tokens of a prefill's row tile.  A workgroup alone on a CU takes about
// 1.7 us a tile of 64 tokens, two 2.5 us (HD 128; the rule is HD 64's too, where a tile takes half
// and three share a CU): `load` row tiles a CU in s slices take about c(load s) / s, c(x) = 1 up to
// one per CU and 3/4 for each begun one from there, with an end that is not full; the slices'
// partial sums and their join cost about 300 load s / tokens of that.
// Measured (us, 40/8 heads of 128): 32 queries over 16384 tokens 430 in one slice, 47 in 16; 511
// queries of each of 4 sequences of up to 16001 493 in one, 443 in 2, 446 in 4; a prompt of 8191 825
// in one, 907 in 2.  Order-preserving as bits: it is positive.
__host__ __device__ inline float slices_cost(float load, int s, float tokens) {
#pragma clang fp contract(off)  // every kernel has to choose alike
  const float x = load * (float)s, c = x <= 1.0f ? 1.0f : 0.75f * __builtin_ceilf(x);
  return (c + 0.3f) / (float)s + (s > 1 ? 300.0f * x / tokens : 0.0f);
}

// The slices of a sequence of n tokens: the best number up to a.slices (the best for as many tokens
// as the table addresses) by what its last row tile may see, one for each kSliceUnits tiles begun
// at most: so of 9 tiles there may be slices of 4 and 5, and of a row tile that sees less, empty
// ones.  Over the lanes of a wavefront, a number each.
__device__ inline int prefill_slices(const AttendArgs& a, int n) {
  if (a.slices == 1) return 1;
  int tiles = (n + kTile - 1) / kTile;
  if (a.window > 0) {  // a tile's rows are at most kPrefillRows tokens
    const int64_t most = ((int64_t)a.window + a.sinks + kPrefillRows) / kTile + 3;
    tiles = tiles < most ? tiles : (int)most;
  }
  const int top = (tiles + kSliceUnits - 1) / kSliceUnits;
  const int s = (int)(threadIdx.x & 31) + 1;
  // the cost's upper bits and the number, the less the better
  int key = (__float_as_int(slices_cost(a.load, s, (float)(tiles * kTile))) & ~31) | (s - 1);
  key = s == 1 || (s <= a.slices && s <= top) ? 0x7fffffff - key : 0;
  return ((0x7fffffff - lane63(wave_prefix(key, Max()))) & 31) + 1;
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

__device__ inline bool sees(int j, int pos, int window, int sinks) {
  return j <= pos && (window <= 0 || j < sinks || j > pos - window);
}

hipError_t launch_append(const Geo& g, const AppendArgs& a, int batch, hipStream_t s);
hipError_t launch_read(const Geo& g, const Pool& p, const int32_t* starts, const int32_t* ends,
                       const int32_t* tables, int batch, int total, void* k, void* v, int type,
                       hipStream_t s);
hipError_t launch_decode(const Geo& g, const AttendArgs& a, int nb, hipStream_t s);
hipError_t launch_decay(const Geo& g, const AttendArgs& a, hipStream_t s);  // of a call of no queries
hipError_t launch_prefill(const Geo& g, const AttendArgs& a, hipStream_t s);
// (query, head) rows of a workgroup of the prefill's merge: a thread per 4 channels, 256 threads
constexpr int merge_log2(int hd) { return hd == 128 ? 3 : 4; }
hipError_t launch_evict(const Geo& g, const float* w, const int32_t* lens, const int32_t* tables,
                        int batch, int keep, int sink, int recent, int32_t* tables_out,
                        int32_t* lens_out, float* w_out, int32_t* evicted, hipStream_t s);

}  // namespace q8
}  // namespace jacq
