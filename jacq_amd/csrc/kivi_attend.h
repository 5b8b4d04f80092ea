// kivi_attend.h -- attention of chunks of queries over the int4 cache, and its read-back: arguments,
// spans, dequantisation.
#pragma once

#include "attend_common.h"
#include "kivi_common.h"

namespace jacq {

struct KiviPool {
  const uint8_t* k_code;
  const uint16_t* k_scale;
  const uint16_t* k_zero;
  const uint8_t* v_code;
  const uint16_t* v_scale;
  const uint16_t* v_zero;
  const uint16_t* k_scr;
  const uint16_t* v_scr;
};

struct KiviAttendArgs {
  KiviPool pool;
  const uint16_t* q;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* tables;
  void* o;
  float* lse;             // null: not wanted
  float* row_lse;         // null
  int64_t q_stride;
  int q_bf16, o_type;     // o_type: kFp16, kBf16, kFp32
  int batch, total_q, max_q;
  int window, sinks;      // window 0: none
  int causal;             // 0: every query sees every token
  int above, upto;        // a launch takes the sequences of more queries than the one, at most the other
  float scale;            // log2(e) included
  // split pieces
  float* part_ml;         // few queries: [target + segments][rows][2]; prompts: [slices][total_q][nh][2]
  float* part_acc;        // the same [HD]
  int32_t* plan;          // calls of many sequences: [batch + 1] first slices, then their size
  int target;             // slices to aim at; 0: segments stay whole
  int cus;                // compute units
  int rows;               // rows of a segment at most (<= 16 NB)
  int row_blocks;         // row blocks of a sequence at most
  // prompts
  int slices;             // workgroups that share a row tile's tokens, at most
  unsigned tiles, merges; // units of row tiles, and of the merge's (Place)
  int32_t* slots;         // [batch + 1] first tile image of each sequence, then their number, then
                          // (float) the tiles that are a slice's share
  int per_pass;           // tile images of a pass; a sequence's begin in one and may end behind it
  int limit;              // images of a call of one pass, which end in it; else INT32_MAX
  uint8_t* images;        // K [64][HD], then V [HD][64], fp16, as they lie in the LDS
  uint64_t* poison;       // of each image: the tokens whose V is not finite or not there
};

__device__ inline int taken(const KiviAttendArgs& a, int m) { return m > a.above && m <= a.upto ? m : 0; }

__device__ inline int clamp_len(const KiviGeo& g, int n) {
  const int cap = g.lq + g.residual;
  return n < 0 ? 0 : n > cap ? cap : n;
}

// The units of kGroup tokens that the queries of a sequence of n tokens may see, in order: the
// sinks', then the window's; int4 groups before `old`, fp16 rows of the residual window from there.
struct KiviSpan {
  int n;        // tokens
  int first;    // the lowest position of a query (may be negative)
  int old;      // tokens in int4
  int w0;       // first unit of the window
  int ns;       // units of the sinks before it
  int units;    // of a segment, at least 1 (a segment without tokens still writes its zeros)
  __device__ int tile_of(int u) const { return u < ns ? u : w0 + u - ns; }
};

__device__ inline KiviSpan make_span(const KiviGeo& g, const KiviAttendArgs& a, int n, int all) {
  KiviSpan s;
  int residual;
  s.n = n;
  s.first = a.causal ? n - all : n - 1;
  decode_window(g, n, &s.old, &residual);
  const int tiles = (n + kGroup - 1) / kGroup;
  s.w0 = s.ns = 0;
  if (a.window > 0 && s.first >= a.window) {
    s.w0 = (s.first - a.window + 1) / kGroup;
    const int sinks = a.sinks < n ? a.sinks : n;
    s.ns = (sinks + kGroup - 1) / kGroup;
    s.ns = s.ns > s.w0 ? s.w0 : s.ns;
  }
  s.units = s.ns + tiles - s.w0;
  s.units = s.units < 1 ? 1 : s.units;
  return s;
}

// The tiles of kTile tokens that any query of a sequence sees: the sinks', then the window's.
struct KiviTiles {
  int n, old;
  int w0, ns, units;
  __device__ KiviTiles(const KiviGeo& g, const KiviAttendArgs& a, int n_, int first) {
    int residual;
    n = n_;
    decode_window(g, n, &old, &residual);
    const int tiles = (n + kTile - 1) / kTile;
    w0 = ns = 0;
    if (a.window > 0 && first >= a.window) {
      w0 = (first - a.window + 1) / kTile;
      const int sinks = a.sinks < n ? a.sinks : n;
      ns = (sinks + kTile - 1) / kTile;
      ns = ns > w0 ? w0 : ns;
    }
    units = ns + tiles - w0;
  }
  __device__ int tile_of(int u) const { return u < ns ? u : w0 + u - ns; }
  __device__ int unit_of(int tile) const { return tile < ns ? tile : tile - w0 + ns; }
};

// Tiles that a row tile of a sequence goes through, about: half of its own queries' are behind its rows.
__device__ inline float row_tiles_units(const KiviAttendArgs& a, const KiviTiles& t, int m, int all) {
#pragma clang fp contract(off)  // every kernel has to find the same
  float units = (float)t.units;
  if (a.window > 0) {
    const float most = ((float)a.window + (float)a.sinks + (float)kPrefillRows) / (float)kTile + 2.0f;
    units = units < most ? units : most;
  } else if (a.causal) {
    units -= ((float)all - 0.5f * (float)m) / (float)kTile;
  }
  return units < 1.0f ? 1.0f : units;
}

// Workgroups that share the tokens of each of a sequence's row tiles.
__device__ inline int kivi_slices(const KiviAttendArgs& a, const KiviTiles& t, int m, int all) {
  if (a.slices == 1) return 1;
  const float share = __int_as_float(a.slots[a.batch + 1]);
  const int n = (int)__builtin_ceilf(row_tiles_units(a, t, m, all) / share);
  return n < 1 ? 1 : n > a.slices ? a.slices : n;
}
__device__ inline int row_slices(const KiviGeo& g, const KiviAttendArgs& a, const Place& p) {
  return kivi_slices(a, KiviTiles(g, a, p.n, a.causal ? p.n - p.all : p.n - 1), p.m, p.all);
}

// A query sees its own token at least, or in no order all of them.
__device__ inline bool sees_any(const KiviGeo&, const KiviAttendArgs& a, int n, int first, int tok) {
  return (a.causal ? first + tok : n - 1) >= 0;
}

// A mean of fp16 values is one, but the sum of the weights that they are multiplied by, each rounded to
// fp16, may be a 2^-11th above the sum l that divides it: beside 65504 that is beyond fp16.  An instruction a
// value (a sum that is NaN comes with an l that is).
__device__ inline float bounded(const KiviGeo&, float sum, float l) {
  return __builtin_amdgcn_fmed3f(sum, -65504.0f * l, 65504.0f * l);
}

template <>
struct SpanOf<KiviGeo> {
  typedef KiviSpan type;
};

// ---- codes to fp16 ----
// A code in a byte of its own is, as e4m3, code x 2^-9 (the format's steps from 0 to 16 x 2^-9 are
// even), so the conversion instruction with scale 2^9 gives two codes as exact fp16.  A value is
// code * scale + zero, rounded to fp16 once: off by at most half a step, 2^-11 of it.

struct Nibbles {
  uint32_t even, odd;  // a dword's codes 0, 2, 4, 6 and 1, 3, 5, 7, a byte each
  __device__ Nibbles(uint32_t w) : even(w & 0x0f0f0f0fu), odd(w >> 4 & 0x0f0f0f0fu) {}
};
__device__ inline h2 codes_lo(uint32_t bytes) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)bytes, 512.0f, false);
}
__device__ inline h2 codes_hi(uint32_t bytes) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)bytes, 512.0f, true);
}
__device__ inline h2 fma2(h2 c, h2 s, h2 z) { return __builtin_elementwise_fma(c, s, z); }
__device__ inline h2 pair(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ inline uint32_t bits(h2 x) { return __builtin_bit_cast(uint32_t, x); }

// 8 channels of a token (one dword), scales and zeros as they lie: the channels in their order.
__device__ inline h8 values8(uint32_t w, u4 s, u4 z) {
  const Nibbles n(w);
  const uint32_t lo = __builtin_amdgcn_perm(n.odd, n.even, 0x05010400u);  // codes 0, 1, 2, 3
  const uint32_t hi = __builtin_amdgcn_perm(n.odd, n.even, 0x07030602u);  // 4, 5, 6, 7
  h8 r;
  r.s01 = fma2(codes_lo(lo), pair(s.x), pair(z.x));
  r.s23 = fma2(codes_hi(lo), pair(s.y), pair(z.y));
  r.s45 = fma2(codes_lo(hi), pair(s.z), pair(z.z));
  r.s67 = fma2(codes_hi(hi), pair(s.w), pair(z.w));
  return r;
}

// Of 8 channels of two tokens (a dword each) the even or the odd ones, s and z the two tokens' of their 32
// channels: out[c] is channel 2 c + odd of both.
__device__ inline void values8x2(uint32_t a, uint32_t b, int odd, h2 s, h2 z, h2 (&out)[4]) {
  const uint32_t x = odd ? a >> 4 & 0x0f0f0f0fu : a & 0x0f0f0f0fu;
  const uint32_t y = odd ? b >> 4 & 0x0f0f0f0fu : b & 0x0f0f0f0fu;
  const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
  out[0] = fma2(codes_lo(lo), s, z);
  out[1] = fma2(codes_hi(lo), s, z);
  out[2] = fma2(codes_lo(hi), s, z);
  out[3] = fma2(codes_hi(hi), s, z);
}

// The same of 4 channels of two tokens: w has the first token's 16 bits, then the second's.
__device__ inline void values4x2(uint32_t w, int odd, h2 s, h2 z, h2 (&out)[2]) {
  const uint32_t x = odd ? w >> 4 & 0x0f0f0f0fu : w & 0x0f0f0f0fu;
  const uint32_t y = __builtin_amdgcn_perm(0u, x, 0x03010200u);
  out[0] = fma2(codes_lo(y), s, z);
  out[1] = fma2(codes_hi(y), s, z);
}

// A query row's values for the matrix cores, 8 of them in each of N operands, from fp16 or bf16, and
// the scale that goes with them.  fp16 has the bits of bf16 but not its range: a power of two brings
// the row's largest magnitude (`most` joins it over the row's lanes) to 2^14, so values down to 2^-28
// of it keep all their bits.  The scale stays a normal number: for a row of subnormals it may lie below
// fp32's range, and 0 times a masked score's -inf, or what is above it times a score of 0, is NaN.  A finite
// score is below 2^38 before the scale, so at 2^-126 all weights are the 1 that they should be.
template <int N, class F>
__device__ inline float half_row(const u4 (&raw)[N], int bf16, float scale, h8 (&q)[N], F most) {
  if (!bf16) {
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = __builtin_bit_cast(h8, raw[i]);
    return scale;
  }
  auto value = [&](int i, int c) {
    return __uint_as_float(c & 1 ? raw[i][c / 2] & 0xffff0000u : raw[i][c / 2] << 16);
  };
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) big = fmaxf(big, __builtin_fabsf(value(i, c)));
  big = most(big);
  const bool plain = !(big > 0.0f && big < __builtin_inff());
  const int e = plain ? 0 : 14 - __builtin_amdgcn_frexp_expf(big);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) q[i][c] = (_Float16)__builtin_amdgcn_ldexpf(value(i, c), e);
  return fminf(fmaxf(__builtin_amdgcn_ldexpf(scale, -e), 0x1p-126f), 0x1.fffffep127f);
}

// Whether fp16 holds all values of a scale and a zero, the ends being 0 and 15 times the scale from it;
// NaN does not pass, and 65520 is the least that rounds to infinity.
__device__ inline bool holds(float scale, float zero) {
  return __builtin_fabsf(zero) < 65520.0f && __builtin_fabsf(__builtin_fmaf(15.0f, scale, zero)) < 65520.0f;
}

// The largest magnitude of two sets of fp16 pairs as bits, in either half: 0x7c00 and more is no
// finite value.
__device__ inline uint32_t most_bits(uint32_t a, uint32_t b) {
  typedef uint16_t s2 __attribute__((ext_vector_type(2)));
  const s2 x = __builtin_bit_cast(s2, a & 0x7fff7fffu), y = __builtin_bit_cast(s2, b & 0x7fff7fffu);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}
__device__ inline uint32_t either_half(uint32_t x) { return (x >> 16) > (x & 0xffffu) ? x >> 16 : x & 0xffffu; }

hipError_t launch_attend_few(const KiviGeo& g, const KiviAttendArgs& a, int nb, hipStream_t s);
// Prompts: `passes` times the images of some sequences and their row tiles, then the slices' merge.
hipError_t launch_attend_prompt(const KiviGeo& g, const KiviAttendArgs& a, int passes, hipStream_t s);
hipError_t launch_kivi_read(const KiviGeo& g, const KiviPool& p, const int32_t* starts,
                            const int32_t* ends, const int32_t* tables, int batch, int total, void* k,
                            void* v, int type, hipStream_t s);
// Workgroups of the prompts' kernel that a CU holds: what its registers and, with V in one buffer, its LDS
// (48 and 24 KB) allow.  A prompt of 8191 tokens, 40/8 heads of 128, takes the kernel 639 us with three, 696
// with two and V in two buffers.
constexpr int prompt_groups(int hd) { return hd == 128 ? 3 : 4; }
// Workgroups of the few-query kernel that a CU holds: what its registers allow.  One more of HD 128 with 32
// rows does not fit (260 bytes of them would lie in memory).
constexpr int few_groups(int hd, int nb) { return hd == 64 ? 5 - nb : 4 - nb; }

}  // namespace jacq
