// attend_common.h -- what the attention kernels of the 8-bit and of the int4 cache share: softmax
// constants, how a call's queries and tokens are cut among workgroups, and how the pieces are joined.
//
// The functions take a cache's geometry G and arguments A by their fields: g.nh, nkv, gqa; a.cu, lens,
// q..., batch, total_q, max_q, window, sinks, o, o_type, lse, row_lse, part_ml, part_acc, plan, target,
// cus, rows, row_blocks, slices, load.  clamp_len(g, n), make_span(g, a, n, all) and slice_units(a, ...)
// are the cache's own.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jacq {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
// element types of queries and outputs, as the C ABIs number them
constexpr int kFp16 = 0, kBf16 = 1, kFp32 = 2;
constexpr int kTile = 64;            // tokens per step of the attention kernels
constexpr int kRowsLog2 = 7;
constexpr int kPrefillRows = 1 << kRowsLog2;  // query rows of a workgroup of the prefill kernel
constexpr int kSliceUnits = 8;       // tiles of one of its slices, about, at least (prefill_slices)
constexpr int kMaxSlices = 32;       // of its slices at most
constexpr int kSliceWaves = 4;       // wavefronts of a workgroup of the few-query kernels: they share a
                                     // slice, unit by unit
// (query, head) rows of a workgroup of merge_slices: a thread per 4 channels, 256 threads
constexpr int merge_log2(int hd) { return hd == 128 ? 3 : 4; }
constexpr float kLog2e = 1.4426950408889634f;
// The weights 2^(t - m) that are rounded to fp16, the type that the matrix cores take at full rate
// with the most bits: m moves to kLift below a row's largest t, and only where that has passed m by
// kSlack more.  So they end at 2^15, the largest so far is at least 2^7, and the others keep 11 bits
// (half a step: 2^-11 of them) down to 2^-14, and are off by at most 2^-25 below.  O loses at most n
// 2^-32 of the largest |v| in the heaviest's block to that; the sum that divides it is of the
// unrounded weights, in fp32.
constexpr float kLift = 7.0f;
constexpr float kSlack = 8.0f;

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

// How many of a sequence's m queries a launch takes: all, unless the cache's own overload says otherwise.
template <class A>
__device__ inline int taken(const A&, int m) {
  return m;
}

// Queries of sequence b: rows [q0, q0 + m) of Q, whatever the table of offsets holds.  m is at most
// max_q; `all` are the sequence's own, which its last tokens are.
template <class A>
__device__ inline void queries_of(const A& a, int b, int* q0, int* m, int* all) {
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
  *m = taken(a, hi - lo > a.max_q ? a.max_q : hi - lo);
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
template <class G, class A>
__device__ inline Place place_of(const G& g, const A& a, int unit, int per, int log2) {
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
  const int m = taken(a, hi - lo > a.max_q ? a.max_q : hi - lo);
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
template <class A>
__device__ inline int prefill_slices(const A& a, int n) {
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

__device__ inline bool sees(int j, int pos, int window, int sinks) {
  return j <= pos && (window <= 0 || j < sinks || j > pos - window);
}

// ---- prompts ----

// LDS writes are done, loads from memory may be in flight.
__device__ inline void turn() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The value of the lane 32 on (or back).
__device__ inline float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}

// 4 values of O, in its type.
template <class A>
__device__ inline void store4(const A& a, int64_t at, f4 x) {
  if (a.o_type == kFp32) {
    *(f4*)((float*)a.o + at) = x;
    return;
  }
  const bool bf = a.o_type == kBf16;
  const uint32_t x0 = bf ? f2bf(x.x) : f2h_(x.x), x1 = bf ? f2bf(x.y) : f2h_(x.y);
  const uint32_t x2 = bf ? f2bf(x.z) : f2h_(x.z), x3 = bf ? f2bf(x.w) : f2h_(x.w);
  *(u2*)((uint16_t*)a.o + at) = u2{x0 | x1 << 16, x2 | x3 << 16};
}

// Whether query `tok` of a sequence of n tokens, whose first one stands at position `first`, sees any: then
// weights whose sum is 0 are of scores that all are -inf.  Of a cache without a rule of its own they are
// taken as a row's that sees nothing.
template <class G, class A>
__device__ inline bool sees_any(const G&, const A&, int /*n*/, int /*first*/, int /*tok*/) {
  return false;
}

// What a row's weighted sums are multiplied by: 1 / l; where the row sees nothing 0, and where all that it
// sees weighs nothing NaN, as 0 / 0.
__device__ inline float over_sum(float l, bool sees) {
  return l != 0.0f ? 1.0f / l : sees ? __builtin_nanf("") : 0.0f;
}

// A weighted sum of values, bounded by the largest value times the sum l of the weights; of a cache without a
// rule of its own there is no largest value.
template <class G>
__device__ inline float bounded(const G&, float sum, float /*l*/) {
  return sum;
}

// Bits 0 to n - 1; n in any range.
__device__ inline uint64_t low_bits(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << n) - 1;
}

// Joins the slices of every row, in their order: a thread per 4 channels, 256 a workgroup.  row_slices is
// the cache's own rule.
template <int HD, class G, class A>
__device__ inline void merge_slices(const G& g, const A& a) {
  static_assert(256 / (HD / 4) == 1 << merge_log2(HD), "rows of a workgroup");
  const Place p = place_of(g, a, blockIdx.x, g.nh, merge_log2(HD));
  const int slices = uniform(row_slices(g, a, p));
  if (slices == 1 || p.at < 0) return;
  const int64_t i = (int64_t)p.at * 256 + threadIdx.x;
  const int ch = (int)(i % (HD / 4)) * 4;
  if (i / (HD / 4) >= (int64_t)p.m * g.nh) return;
  const int64_t at = (int64_t)p.q0 * g.nh + i / (HD / 4), rows = (int64_t)a.total_q * g.nh;
  float mx = kNegInf, l = 0.0f;
  f4 acc = {0, 0, 0, 0};
  for (int s = 0; s < slices; ++s) {
    const float pm = a.part_ml[2 * (s * rows + at)], pl = a.part_ml[2 * (s * rows + at) + 1];
    const f4 pa = *(const f4*)(a.part_acc + (s * rows + at) * HD + ch);
    const float to = fmaxf(mx, pm);
    // a part without a maximum saw nothing, or only NaN: l tells
    const float f0 = mx == kNegInf ? 1.0f : exp2_(mx - to);
    const float f1 = pm == kNegInf ? 1.0f : exp2_(pm - to);
    acc = acc * f0 + pa * f1;
    l = l * f0 + pl * f1;
    mx = to;
  }
  const float inv = over_sum(l, sees_any(g, a, p.n, p.n - p.all, (int)(i / (HD / 4)) / g.nh));
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = bounded(g, acc[c], l);
  store4(a, at * HD + ch, acc * inv);
  if (a.lse && ch == 0) a.lse[at] = l == 0.0f ? kNegInf : (mx + log2_(l)) / kLog2e;
}

// ---- a few queries per sequence ----

// One segment's place: sequence, kv head, row block, and its units' span.  Each cache has a Span of
// its own (SpanOf of its geometry), which make_span finds for a sequence of n tokens whose queries
// are `all`: span.units units, and span.first the position of the first query.
template <class G>
struct SpanOf;
template <class G>
struct Segment {
  int b, h, rb;
  int q0, m;      // its sequence's first query and number of queries
  int nrows;      // of this block
  typename SpanOf<G>::type span;
};

template <class A>
__device__ inline void store_row(const A& a, int64_t at, const float* x, int n) {
  if (a.o_type == kFp32) {
    for (int i = 0; i < n; i += 4) *(f4*)((float*)a.o + at + i) = *(const f4*)(x + i);
    return;
  }
  for (int i = 0; i < n; i += 2) {
    const uint32_t lo = a.o_type == kBf16 ? f2bf(x[i]) : f2h_(x[i]);
    const uint32_t hi = a.o_type == kBf16 ? f2bf(x[i + 1]) : f2h_(x[i + 1]);
    *(uint32_t*)((uint16_t*)a.o + at + i) = lo | hi << 16;
  }
}

// O and lse of a row from sum(w v), sum(w / vs) and the maximum that w refers to.
template <class G, class A>
__device__ inline void finish_row(const G& g, const A& a, const Segment<G>& s, int row, int hd, int ch, float* x, int n, float l, float m) {
  const int r = s.rb * a.rows + row, tok = s.q0 + r / g.gqa, head = s.h * g.gqa + r % g.gqa;
  const float inv = over_sum(l, sees_any(g, a, s.span.n, s.span.first, r / g.gqa));
  for (int i = 0; i < n; ++i) x[i] = bounded(g, x[i], l) * inv;
  store_row(a, ((int64_t)tok * g.nh + head) * hd + ch, x, n);
  if (ch == 0) {
    const float lse = l == 0.0f ? kNegInf : m + log2_(l);
    if (a.lse) a.lse[(int64_t)tok * g.nh + head] = lse / kLog2e;
    if (a.row_lse) a.row_lse[(int64_t)tok * g.nh + head] = lse;
  }
}

template <int ROWS, class G, class A, class S>
__device__ inline void sequence_span(const G& g, const A& a, int b, int* q0, int* m, S* span,
                                     int* blocks) {
  int all;
  queries_of(a, b, q0, m, &all);
  const int n = clamp_len(g, a.lens[b]);
  *span = make_span(g, a, n, all);
  *blocks = (*m * g.gqa + ROWS - 1) / ROWS;
}

// How the call's segments are cut: into slices of about `size` units each, at most a.target of
// them more than there are segments.  A sequence's slices are numbered from `before` on, kv head
// by kv head fastest, then row block, then slice.
struct Slices {
  int size;
  int b;
  int before;
};

template <class S>
__device__ inline int slices_of(const S& s, int size) { return (s.units + size - 1) / size; }

// Units of each of the n slices but the last: equal, in whole rounds of the wavefronts too (never
// more than the size they were counted by, so the last has some left).
template <class S>
__device__ inline int even_units(const S& s, int n) {
  const int u = (s.units + n - 1) / n;
  return n == 1 ? u : (u + kSliceWaves - 1) / kSliceWaves * kSliceWaves;
}

// The same of a cut that plan_cut left: 64 places a step.
template <class A>
__device__ inline Slices planned(const A& a, int lane, int want, int b) {
  const int size = uniform(a.plan[a.batch + 1]);
  if (want < 0) return {size, b, uniform(a.plan[b])};
  if (want >= uniform(a.plan[a.batch])) return {size, a.batch, 0};
  // the last sequence whose first slice is not behind `want`: one without slices is not the last
  int at = 0;
  for (int n = a.batch; n > 1;) {
    const int step = (n + 63) / 64, i = lane * step;
    const uint64_t upto = __ballot(i < n && a.plan[at + (i < n ? i : 0)] <= want);
    const int skip = (__popcll(upto) - 1) * step;
    at += skip;
    n = step < n - skip ? step : n - skip;
  }
  return {size, at, uniform(a.plan[at])};
}

// The cut, and the sequence that has slice `want` (b >= batch: none), or, with want < 0, the place
// of sequence `b`.  slice_units is the cache's own rule.  Over the lanes of each wavefront alike, a sequence each.
template <int ROWS, class G, class A>
__device__ inline Slices cut(const G& g, const A& a, int lane, int want, int b) {
#pragma clang fp contract(off)
  if (a.plan) return planned(a, lane, want, b);
  // the sums are fp32: they choose the size, alike in every wavefront and kernel, and no more
  float u = 0.0f, n = 0.0f;
  int q0, m, blocks = 0, most = 1;
  typename SpanOf<G>::type sp;
  if (lane < a.batch) {
    sequence_span<ROWS>(g, a, lane, &q0, &m, &sp, &blocks);
    n = (float)(blocks * g.nkv);
    u = (float)sp.units * n;
    most = blocks ? sp.units : 1;
  }
  const float total = __int_as_float(lane63(wave_prefix(__float_as_int(u), SumF())));
  const float segments = __int_as_float(lane63(wave_prefix(__float_as_int(n), SumF())));
  const int size = uniform(slice_units(a, total, segments, lane63(wave_prefix(most, Max()))));
  const int count = lane < a.batch ? slices_of(sp, size) * blocks * g.nkv : 0;
  const int inc = wave_prefix(count, Sum());
  if (want < 0) return {size, b, __builtin_amdgcn_readlane(inc - count, uniform(b))};
  if (const uint64_t past = __ballot(inc > want && count > 0)) {
    const int l = __builtin_ctzll(past);
    return {size, l, __builtin_amdgcn_readlane(inc - count, l)};
  }
  return {size, a.batch, 0};
}

// The segment of this workgroup, and its units of it: target > 0: slice blockIdx.x of the cut; else
// the segment blockIdx.x = (sequence, row block, kv head) whole.  False: none.
template <int ROWS, class G, class A>
__device__ inline bool place_slice(const G& g, const A& a, int lane, Segment<G>& s, int& u0, int& u1,
                                   bool& whole) {
  int blocks;
  u0 = 0;
  whole = true;
  if (a.target) {
    const Slices c = cut<ROWS>(g, a, lane, blockIdx.x, 0);
    if (c.b >= a.batch) return false;
    s.b = c.b;
    sequence_span<ROWS>(g, a, s.b, &s.q0, &s.m, &s.span, &blocks);
    int x = blockIdx.x - c.before;
    s.h = uniform(x % g.nkv);
    x /= g.nkv;
    s.rb = uniform(x % blocks);
    const int z = uniform(x / blocks), n = uniform(slices_of(s.span, c.size));
    const int each = uniform(even_units(s.span, n));
    u0 = z * each;
    u1 = u0 + each < s.span.units ? u0 + each : s.span.units;
    whole = n == 1;
  } else {
    s.b = blockIdx.x / (g.nkv * a.row_blocks);
    s.h = blockIdx.x % g.nkv;
    s.rb = blockIdx.x / g.nkv % a.row_blocks;
    sequence_span<ROWS>(g, a, s.b, &s.q0, &s.m, &s.span, &blocks);
    if (s.rb >= blocks) return false;
    u1 = s.span.units;
  }
  const int left = s.m * g.gqa - s.rb * ROWS;
  s.nrows = left < ROWS ? left : ROWS;
  return true;
}

// Joins the wavefronts' parts of a slice: sum(w v) in red[wave][row][channel] and, in ml, the maximum
// that w refers to and the sum of w; to O, or to the slice's place in the workspace.  `rows` of the
// segment's from row0 on.
template <int HD, class G, class A, int ROWS, int LD>
__device__ inline void fold_parts(const G& g, const A& a, const Segment<G>& s, bool whole,
                                  const float (&red)[kSliceWaves][ROWS][LD],
                                  const float (&ml)[kSliceWaves][ROWS][2], int row0, int rows) {
  constexpr int PER = HD / 16;  // channels of a thread
  for (int i = threadIdx.x; i < rows * 16; i += 64 * kSliceWaves) {
    const int row = i / 16, ch = i % 16 * PER;
    float mm = kNegInf, l = 0.0f;
#pragma unroll
    for (int v = 0; v < kSliceWaves; ++v) mm = fmaxf(mm, ml[v][row][0]);
    float x[PER];
#pragma unroll
    for (int c = 0; c < PER; ++c) x[c] = 0.0f;
#pragma unroll
    for (int v = 0; v < kSliceWaves; ++v) {
      // a part without a maximum saw nothing, or only NaN: l tells
      const float mv = ml[v][row][0];
      const float f = mv == kNegInf ? 1.0f : exp2_(mv - mm);
      l += ml[v][row][1] * f;
#pragma unroll
      for (int c = 0; c < PER; ++c) x[c] += red[v][row][ch + c] * f;
    }
    if (whole) {
      finish_row(g, a, s, row0 + row, HD, ch, x, PER, l, mm);
    } else {
      const int64_t at = (int64_t)blockIdx.x * a.rows + row0 + row;
#pragma unroll
      for (int c = 0; c < PER; c += 4) *(f4*)(a.part_acc + at * HD + ch + c) = *(f4*)(x + c);
      if (ch == 0) {
        a.part_ml[at * 2] = mm;
        a.part_ml[at * 2 + 1] = l;
      }
    }
  }
}

// The cut of many sequences, once for the call.  One workgroup of 1024.
template <int ROWS, class G, class A>
__device__ inline void plan_cut(const G& g, const A& a) {
  __shared__ float units[16], segments[16];
  __shared__ int longest[16], sums[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int q0, m, blocks;
  typename SpanOf<G>::type sp;
  float u = 0.0f, n = 0.0f;
  int most = 1;
  for (int b = tid; b < a.batch; b += 1024) {
    sequence_span<ROWS>(g, a, b, &q0, &m, &sp, &blocks);
    n += (float)(blocks * g.nkv);
    u += (float)sp.units * (float)(blocks * g.nkv);
    most = blocks && sp.units > most ? sp.units : most;
  }
  u = __int_as_float(lane63(wave_prefix(__float_as_int(u), SumF())));
  n = __int_as_float(lane63(wave_prefix(__float_as_int(n), SumF())));
  most = lane63(wave_prefix(most, Max()));
  if (lane == 0) {
    units[wave] = u;
    segments[wave] = n;
    longest[wave] = most;
  }
  __syncthreads();
  u = n = 0.0f;
  for (int i = 0; i < 16; ++i) {
    u += units[i];
    n += segments[i];
    most = longest[i] > most ? longest[i] : most;
  }
  const int size = uniform(slice_units(a, u, n, most));
  int before = 0;
  for (int base = 0, turn = 0; base < a.batch; base += 1024, turn ^= 1) {
    const int b = base + tid;
    int count = 0;
    if (b < a.batch) {
      sequence_span<ROWS>(g, a, b, &q0, &m, &sp, &blocks);
      count = slices_of(sp, size) * blocks * g.nkv;
    }
    const int inc = wave_prefix(count, Sum());
    if (lane == 63) sums[turn][wave] = inc;
    __syncthreads();  // the other turn's sums have been read by all
    int here = before + inc - count;
    for (int i = 0; i < 16; ++i) {
      here += i < wave ? sums[turn][i] : 0;
      before += sums[turn][i];
    }
    if (b < a.batch) a.plan[b] = here;
  }
  if (tid == 0) {
    a.plan[a.batch] = before;
    a.plan[a.batch + 1] = size;
  }
}

// Joins a segment's slices, in their order.  blockIdx.x: segment.  MANY: of the row blockIdx.y, the
// threads side by side share the slices; else they share the rows, 1024 / HD at a time, with gridDim.y
// workgroups.  256 threads.
template <int HD, int ROWS, bool MANY, class G, class A>
__device__ inline void join_slices(const G& g, const A& a) {
  constexpr int TC = HD / 4;      // threads of a row
  constexpr int PG = 256 / TC;    // rows, or slices, at a time
  const int lane = threadIdx.x & 63;
  Segment<G> s;
  int blocks;
  s.b = blockIdx.x / (g.nkv * a.row_blocks);
  s.h = blockIdx.x % g.nkv;
  s.rb = blockIdx.x / g.nkv % a.row_blocks;
  sequence_span<ROWS>(g, a, s.b, &s.q0, &s.m, &s.span, &blocks);
  if (s.rb >= blocks) return;
  const int left = s.m * g.gqa - s.rb * ROWS;
  s.nrows = left < ROWS ? left : ROWS;
  if (MANY && (int)blockIdx.y >= s.nrows) return;
  const Slices c = cut<ROWS>(g, a, lane, -1, s.b);
  const int n = uniform(slices_of(s.span, c.size));
  if (n == 1) return;
  const int64_t first = c.before + s.rb * g.nkv + s.h;
  const int step = blocks * g.nkv;
  const int grp = threadIdx.x / TC, ch = threadIdx.x % TC * 4;
  auto add = [&](float pm, float pl, f4 pa, float& mm, float& l, f4& acc) {
    const float to = fmaxf(mm, pm);
    const float f0 = mm == kNegInf ? 1.0f : exp2_(mm - to);
    const float f1 = pm == kNegInf ? 1.0f : exp2_(pm - to);
    acc = acc * f0 + pa * f1;
    l = l * f0 + pl * f1;
    mm = to;
  };
  // slices z0, z0 + by, ... of a row, 4 in flight
  auto sum = [&](int row, int z0, int by, float& mm, float& l, f4& acc) {
    for (int z = z0; z < n; z += 4 * by) {
      float pm[4], pl[4];
      f4 pa[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int zz = z + i * by < n ? z + i * by : z;
        const int64_t at = (first + (int64_t)zz * step) * a.rows + row;
        pm[i] = a.part_ml[at * 2];
        pl[i] = a.part_ml[at * 2 + 1];
        pa[i] = *(const f4*)(a.part_acc + at * HD + ch);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (z + i * by < n) add(pm[i], pl[i], pa[i], mm, l, acc);
    }
  };
  if constexpr (!MANY) {
    for (int row = grp + PG * blockIdx.y; row < s.nrows; row += PG * gridDim.y) {
      float mm = kNegInf, l = 0.0f;
      f4 acc = {0, 0, 0, 0};
      sum(row, 0, 1, mm, l, acc);
      float o[4] = {acc.x, acc.y, acc.z, acc.w};
      finish_row(g, a, s, row, HD, ch, o, 4, l, mm);
    }
  } else {
    __shared__ __align__(16) float red[PG][HD];
    __shared__ float ml[PG][2];
    const int row = blockIdx.y;
    float mm = kNegInf, l = 0.0f;
    f4 acc = {0, 0, 0, 0};
    sum(row, grp, PG, mm, l, acc);
    *(f4*)&red[grp][ch] = acc;
    if (ch == 0) {
      ml[grp][0] = mm;
      ml[grp][1] = l;
    }
    __syncthreads();
    if (threadIdx.x >= TC) return;
    mm = kNegInf;
    l = 0.0f;
    acc = f4{0, 0, 0, 0};
    for (int i = 0; i < PG; ++i) add(ml[i][0], ml[i][1], *(const f4*)&red[i][ch], mm, l, acc);
    float o[4] = {acc.x, acc.y, acc.z, acc.w};
    finish_row(g, a, s, row, HD, ch, o, 4, l, mm);
  }
}

}  // namespace jacq
