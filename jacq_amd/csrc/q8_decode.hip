// q8_decode.hip -- attention of a few queries per sequence over the 8-bit cache.
//
// A segment is a (sequence, kv head, block of 16 NB query rows); a row is a
// (query token, head of the kv head's group), so all G heads share every byte.
// Per 64 tokens and wavefront: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32_f16.  The rows of a K operand may be any tokens, so they
// are dealt such that lane quarter kq = lane / 16 gets the scores of 16
// consecutive tokens, its row's P is already the next operand (no shuffle), and
// its V operand is 16 consecutive tokens of a channel: one 16-byte load of
// the transposed V codes.  Codes go from memory to registers to the matrix
// cores, without the LDS.
//
// The V scale is constant over a lane's 16 tokens and enters the exponent:
//   t = s (ks scale log2e) + log2(vs),  w = 2^(t - m),  O = sum(w v) / sum(w / vs)
// so no accumulator needs a scale of its own, and the P that is rounded to fp16
// (kLift has its range; bf16 would be off by 2^-8 of it, fp16 by 2^-11) is at most
// 2^15.  What it may lose is small next to the block of the largest w, so beside a
// block of far larger V scale, not next to the values of a smaller one.
//
// Bound by memory.  Measured (40/8 heads of 128, int8, page 32): 64 sequences of 1024 to 16384
// tokens, one query each, 1.16 GB: 215 us and 5 us for the join, 5.3 TB/s, where a copy of 2 GiB
// runs at 4.96; 4 queries of each of 32 sequences of 1500 to 6007 (32/8 heads, bf16) 47 + 6 us.
// One sequence of 512 tokens (32/4 heads of 64) is latency: 5.5 us, four dependent rounds of
// memory (length, table, codes, and the fold through the LDS).
// Wavefronts a SIMD at HD 128: three of 16 rows, two of 32; the codes of a unit in flight are 64
// registers.  With two and one, 1024 sequences of 100 to 500 tokens took 212 us instead of 178,
// with 8 queries each 489 instead of 288 (32/8 heads); one sequence of 500000 tokens, 4 queries,
// 238 instead of 200 (40/8 heads).
#include "q8_common.h"

namespace jacq {
namespace q8 {

constexpr int kWaves = 4;         // wavefronts of a workgroup: they share a slice, unit by unit
constexpr float kNegInf = -__builtin_inff();

// One segment's place: sequence, kv head, row block, and its units' span.
struct Segment {
  int b, h, rb;
  int q0, m;      // its sequence's first query and number of queries
  int nrows;      // of this block
  Span span;
};

template <int HD, bool E4M3, int NB>
struct Wave {
  static constexpr int KS = HD / 32;  // k-steps of S^T
  static constexpr int KL = HD / 64;  // 16-byte loads of a K row per lane
  static constexpr int DT = HD / 16;  // channel tiles
  const Geo& g;
  const AttendArgs& a;
  int lane, n16, kq;

  h8 q[NB][KS];
  float qs[NB];    // a row's scores are qs times what the matrix cores give (log2(e) included)
  int pos[NB];     // the row's position; below 0 where there is no row
  f4 acc[NB][DT];
  float m[NB], l[NB];
  float group[NB];  // the last tile's, of this lane's 16 tokens

  struct Codes {
    u4 k[4][KL];
    u4 v[DT];
    float ks, vs;
    bool there;  // a page outside the pool reads as NaN
  };

  __device__ Wave(const Geo& g_, const AttendArgs& a_, int lane_)
      : g(g_), a(a_), lane(lane_), n16(lane_ & 15), kq(lane_ >> 4) {}

  __device__ void start(const Segment& s) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = s.rb * 16 * NB + nb * 16 + n16;
      const int tok = row / g.gqa, head = s.h * g.gqa + row % g.gqa;
      const bool ok = tok < s.m;
      pos[nb] = ok ? s.span.first + tok : -1;
      m[nb] = kNegInf;
      l[nb] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[nb][d] = f4{0, 0, 0, 0};
      const uint16_t* src = a.q + (int64_t)(s.q0 + (ok ? tok : 0)) * a.q_stride + head * HD + kq * 16;
      u4 raw[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i)
        raw[i] = ok ? *(const u4*)(src + (i / 2) * 64 + (i & 1) * 8) : u4{0, 0, 0, 0};
      if (a.q_bf16) {
        // fp16 has the bits of bf16 but not its range: a power of two brings the row's largest
        // magnitude to 2^14, so values down to 2^-28 of it keep all their bits.
        float big = 0.0f;
        float f[KS][8];
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t w = raw[i][c / 2];
            f[i][c] = __uint_as_float(c & 1 ? w & 0xffff0000u : w << 16);
            big = fmaxf(big, __builtin_fabsf(f[i][c]));
          }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        const bool plain = !(big > 0.0f && big < __builtin_inff());
        const int e = plain ? 0 : 14 - __builtin_amdgcn_frexp_expf(big);
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int c = 0; c < 8; ++c)
            q[nb][i][c] = (_Float16)__builtin_amdgcn_ldexpf(f[i][c], e);
        qs[nb] = __builtin_amdgcn_ldexpf(a.scale, -e);
      } else {
#pragma unroll
        for (int i = 0; i < KS; ++i) q[nb][i] = __builtin_bit_cast(h8, raw[i]);
        qs[nb] = a.scale;
      }
    }
  }

  // The table's entry for the 16 tokens from t on; it is looked at when its page is loaded, so
  // that nothing waits for it before.
  __device__ int page_of(const Segment& s, int t) const {
    const int last = s.span.nq - 16;  // never past the sequence's own entries
    t = t < last ? t : last;
    return a.tables[(int64_t)s.b * g.max_pages + (t >> g.page_log2)];
  }
  __device__ bool exists(int page) const { return page >= 0 && page < g.num_pages; }
  __device__ uint32_t held(int page) const { return exists(page) ? page : 0; }

  __device__ void pages(const Segment& s, int tile, int& pk, int& pv) const {
    pk = page_of(s, tile * kTile + n16 / 4 * 16);
    pv = page_of(s, tile * kTile + kq * 16);
  }

  // A quantised tile's K codes, its scales and its V codes.  A tile begins a page or lies in one, so
  // where a lane reads in its page is the same for all.
  __device__ void load_k(const Segment& s, int pk, Codes& c) const {
    uint32_t in = (s.h * g.page + (n16 / 4 * 16 & (g.page - 1)) + (n16 & 3)) * HD + kq * 16;
    asm volatile("" : "+v"(in));  // one register over the loop, not a pointer's two
    const uint8_t* k = a.pool.k_code + ((uint64_t)held(pk) * (uint32_t)(g.nkv * g.page * HD) + in);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < KL; ++j) c.k[t][j] = *(const u4*)(k + t * 4 * HD + j * 64);
  }
  __device__ void load_scales(const Segment& s, int pv, Codes& c) const {
    const uint64_t slot = (uint64_t)held(pv) * (uint32_t)g.nkv + (uint32_t)s.h;
    c.ks = a.pool.k_scale[slot];
    c.there = exists(pv);
    c.vs = a.pool.v_scale[slot];
  }
  __device__ void load_v(const Segment& s, int pv, Codes& c) const {
    uint32_t in = (s.h * HD + n16) * g.page + (kq * 16 & (g.page - 1));
    asm volatile("" : "+v"(in));
    const uint8_t* v = a.pool.v_code + ((uint64_t)held(pv) * (uint32_t)(g.nkv * g.page * HD) + in);
#pragma unroll
    for (int d = 0; d < DT; ++d) c.v[d] = *(const u4*)(v + d * 16 * g.page);
  }

  // Scores -> weights -> O^T.  sc: raw scores of this lane's 16 tokens, t0 their first one;
  // tokens from `end` on are not there.  p0, p1: the weights in fp16.
  __device__ void soften(int nb, f4 (&sc)[4], int t0, int end, float ks, float vs,
                         bool masked, h8& p0, h8& p1) {
    const float av = qs[nb] * ks, bv = log2_(vs), ivs = 1.0f / vs;
    float t[16];
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      t[i] = __builtin_fmaf(sc[i / 4][i & 3], av, bv);
      if (masked)
        t[i] = t0 + i < end && sees(t0 + i, pos[nb], a.window, a.sinks) ? t[i] : kNegInf;
      mx = fmaxf(mx, t[i]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__ballot(mx > m[nb] + (kLift + kSlack))) {  // also where m is -inf and mx is not
      const float to = mx > m[nb] + (kLift + kSlack) ? mx - kLift : m[nb];
      const float f = to > m[nb] ? exp2_(m[nb] - to) : 1.0f;
      m[nb] = to;
      l[nb] *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[nb][d] *= f;
    }
    const float base = m[nb] == kNegInf ? 0.0f : m[nb];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = exp2_(t[i] - base);
      sum += w;
      if (i < 8) p0[i] = (_Float16)w;
      else p1[i - 8] = (_Float16)w;
    }
    const float part = sum == 0.0f ? 0.0f : sum * ivs;  // a scale that nothing sees may be any
    l[nb] += part;
    group[nb] = base + log2_(part);
  }

  // The base-2 logarithms of the weight of this lane's 16 tokens from t0 on, for the block weights.
  // In fp32, as the row's own that the weights kernel takes from them: the weight is of the row's
  // whole sum, which is not known yet, and a logarithm needs no rescaling when the maximum moves.  Of
  // a magnitude of up to 2^8, it leaves a weight within 2^-15 of itself.
  __device__ void store_group(const Segment& s, int t0, int end) const {
    if (!a.weights || t0 >= end) return;
    const int64_t seg = ((int64_t)s.b * g.nkv + s.h) * a.row_blocks + s.rb;
    float* dst = a.group_lse + (seg * a.groups + (t0 >> 4)) * a.rows;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (nb * 16 + n16 < s.nrows) dst[nb * 16 + n16] = group[nb];
  }

  __device__ bool needs_mask(const Segment& s, int t0, int end) const {
    // uniform: the tile's 64 tokens are all there and every row sees them
    const int first = s.span.first + s.rb * 16 * NB / g.gqa;
    const int last = s.span.first + (s.rb * 16 * NB + s.nrows - 1) / g.gqa;
    return t0 + kTile > end || t0 + kTile - 1 > first ||
           (a.window > 0 && t0 <= last - a.window && t0 + kTile > a.sinks);
  }

  // No row sees the 16 tokens from t on, as their windows begin later: their page may be any, and
  // its e4m3 codes NaN, which a weight of 0 would not take out.
  __device__ bool before_window(const Segment& s, int t) const {
    const int first = s.span.first + s.rb * 16 * NB / g.gqa;
    return t + 15 <= first - a.window && t >= a.sinks;
  }

  __device__ void scores(const Codes& c, f4 (&sc)[NB][4]) const {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sc[nb][t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const u4 w = c.k[t][i / 2];
        const h8 k = i & 1 ? codes8<E4M3>(w.z, w.w) : codes8<E4M3>(w.x, w.y);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          sc[nb][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[nb][i], sc[nb][t], 0, 0, 0);
      }
    }
  }

  __device__ void values(const Codes& c, const h8 (&p)[NB][2]) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const h8 v0 = codes8<E4M3>(c.v[d].x, c.v[d].y), v1 = codes8<E4M3>(c.v[d].z, c.v[d].w);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        acc[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[nb][0], acc[nb][d], 0, 0, 0);
        acc[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[nb][1], acc[nb][d], 0, 0, 0);
      }
    }
  }

  // The tail: fp16 rows [nq, n), at most P of them.  Once per segment; V is gathered value by
  // value.
  __device__ void tail(const Segment& s) {
    const int rows = s.span.n - s.span.nq;
    if (rows <= 0) return;
    const int64_t base = ((int64_t)s.b * g.nkv + s.h) * g.page * HD;
    const uint16_t* k = a.pool.k_tail + base + kq * 16;
    const uint16_t* v = a.pool.v_tail + base + n16;
    f4 sc[NB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      int r = n16 / 4 * 16 + t * 4 + (n16 & 3);
      r = r < rows ? r : rows - 1;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sc[nb][t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const h8 kk = *(const h8*)(k + r * HD + (i / 2) * 64 + (i & 1) * 8);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          sc[nb][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[nb][i], sc[nb][t], 0, 0, 0);
      }
    }
    h8 p[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      soften(nb, sc[nb], s.span.nq + kq * 16, s.span.n, 1.0f, 1.0f, true, p[nb][0], p[nb][1]);
    store_group(s, s.span.nq + kq * 16, s.span.n);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      h8 vv[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = kq * 16 + i;
        // what lies behind the last token is not read: it may be anything
        const uint16_t x = r < rows ? v[r * HD + d * 16] : (uint16_t)0;
        vv[i / 8][i & 7] = __builtin_bit_cast(_Float16, x);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        acc[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[0], p[nb][0], acc[nb][d], 0, 0, 0);
        acc[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[1], p[nb][1], acc[nb][d], 0, 0, 0);
      }
      if (NB == 2 || d & 1) __builtin_amdgcn_sched_barrier(0);  // few loads at a time: registers
    }
  }

  // Units u0, u0 + kWaves, ... below u1.  One set of code registers: the next tile's K is
  // loaded when this one's scores are done, its V when this one's is used up.
  __device__ void units(const Segment& s, int u0, int u1) {
    if (u0 >= u1) return;
    const Span& sp = s.span;
    const int quant = sp.ns + sp.tiles - sp.w0;  // units of quantised tiles
    const int e = u1 < quant ? u1 : quant;
    if (u0 < e) {
      Codes c;
      int pk, pv, nk = 0, nv = 0, tile = sp.tile_of(u0);
      pages(s, tile, pk, pv);
      load_k(s, pk, c);
      load_scales(s, pv, c);
      load_v(s, pv, c);
      if (u0 + kWaves < e) pages(s, sp.tile_of(u0 + kWaves), nk, nv);
      for (;;) {
        const int next = u0 + kWaves < e ? sp.tile_of(u0 + kWaves) : -1;
        const int t0 = tile * kTile;
        const bool masked = needs_mask(s, t0, sp.nq);
        f4 sc[NB][4];
        scores(c, sc);
        const float ks = c.there ? c.ks : __builtin_nanf(""), vs = c.vs;
        // a page outside the pool reads as page 0, whose e4m3 codes may be NaN: as before a window
        if (E4M3 && masked && (!c.there || (a.window > 0 && before_window(s, t0 + kq * 16))))
#pragma unroll
          for (int d = 0; d < DT; ++d) c.v[d] = u4{0, 0, 0, 0};
        if (next >= 0) load_k(s, nk, c);
        h8 p[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          soften(nb, sc[nb], t0 + kq * 16, sp.nq, ks, vs, masked, p[nb][0], p[nb][1]);
        values(c, p);
        u0 += kWaves;
        if (next < 0) break;
        load_scales(s, nv, c);
        load_v(s, nv, c);
        // behind the loads: what is loaded behind a store waits for it too (256 sequences of 100 to
        // 4000 tokens, 32/8 heads of 128: 241 us against 246)
        store_group(s, t0 + kq * 16, sp.nq);
        if (u0 + kWaves < e) pages(s, sp.tile_of(u0 + kWaves), nk, nv);
        tile = next;
      }
      store_group(s, tile * kTile + kq * 16, sp.nq);
    }
    if (u0 < u1) tail(s);  // the unit behind the quantised ones
  }
};

__device__ inline void store_row(const AttendArgs& a, int64_t at, const float* x, int n) {
  if (a.o_type == JACQ_Q8_FP32) {
    for (int i = 0; i < n; i += 4) *(f4*)((float*)a.o + at + i) = *(const f4*)(x + i);
    return;
  }
  for (int i = 0; i < n; i += 2) {
    const uint32_t lo = a.o_type == JACQ_Q8_BF16 ? f2bf(x[i]) : f2h_(x[i]);
    const uint32_t hi = a.o_type == JACQ_Q8_BF16 ? f2bf(x[i + 1]) : f2h_(x[i + 1]);
    *(uint32_t*)((uint16_t*)a.o + at + i) = lo | hi << 16;
  }
}

// O and lse of a row from sum(w v), sum(w / vs) and the maximum that w refers to.
__device__ inline void finish_row(const Geo& g, const AttendArgs& a, const Segment& s, int row,
                                  int hd, int ch, float* x, int n, float l, float m) {
  const int r = s.rb * a.rows + row, tok = s.q0 + r / g.gqa, head = s.h * g.gqa + r % g.gqa;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int i = 0; i < n; ++i) x[i] *= inv;
  store_row(a, ((int64_t)tok * g.nh + head) * hd + ch, x, n);
  if (ch == 0) {
    const float lse = l == 0.0f ? kNegInf : m + log2_(l);
    if (a.lse) a.lse[(int64_t)tok * g.nh + head] = lse / kLog2e;
    if (a.row_lse) a.row_lse[(int64_t)tok * g.nh + head] = lse;
  }
}

template <int ROWS>
__device__ inline void sequence_span(const Geo& g, const AttendArgs& a, int b, int* q0, int* m,
                                     Span* span, int* blocks) {
  int all;
  queries_of(a, b, q0, m, &all);
  const int n = clamp_len(g, a.lens[b]);
  *span = Span(g, n, n - all, a.window, a.sinks);
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

__device__ inline int slices_of(const Span& s, int size) { return (s.units + size - 1) / size; }

// Units of a slice, from the call's units, its segments and the longest one's units.
//  - Uncut, if that takes no longer: a workgroup alone on a CU needs about 0.4 us a unit (HD 128,
//    whose rule is HD 64's too), the memory 0.8 us a unit and CU, a cut call about 2 us more; and
//    where segments outnumber CUs only if they are about equally long and, with up to 16 rows, fill
//    the CUs about evenly.  40/8
//    heads of 128, uncut against cut (us): 32 sequences of 2048 tokens 27.8 against 29.5, 64 48.2
//    against 50.3, 64 of 4096 103 against 110; 16 of 1000 22.3 against 18.1, of 2000 30.2 against
//    25.7, of 4096 41.6 against 31.7; 64 of 1024 to 16384 267 against 235; one of 4096 35.3 against
//    12.6; 48 with windows of 4096, 32/8 heads, 91 against 87; 4 queries of 48 of 3000 to 3500 77
//    against 91.
//  - Else as many slices as the chip holds workgroups, once or twice (a.target), where a segment's
//    last slice counts half, so that few are left for another round; of 4 to 16 units where there is
//    less work, and whole rounds of the workgroup's wavefronts.  A fixed 4 a CU took, us: 3 sequences
//    of 20001 to 65535, 64/8 heads 58 against 53; 24 of 4096 to 12289, 40/8 heads, with block weights
//    106 against 100; 16 of 1000 to 8000, 32/32 heads 117 against 110.
__device__ inline int slice_units(const AttendArgs& a, float all, float segments, int longest) {
#pragma clang fp contract(off)  // the decode and the join have to find the same size
  const float cus = (float)a.cus;
  const bool even = a.rows > 16 || segments >= 0.8f * cus * __builtin_ceilf(segments / cus);
  if ((float)longest <= 1.4f * all / cus + 4.0f &&
      (segments <= cus || (even && all >= 0.75f * segments * (float)longest)))
    return longest;
  const int fair = (int)(all / cus) + 1;  // one slice a CU
  const int few = fair < 4 ? 4 : fair > 16 ? 16 : fair;
  const float fit = (float)a.target - 0.5f * segments, half = 0.5f * (float)a.target;
  const int many = (int)(all / (fit > half ? fit : half)) + 1;
  return ((many > few ? many : few) + kWaves - 1) / kWaves * kWaves;
}

// Units of each of the n slices but the last: equal, in whole rounds of the wavefronts too (never
// more than the size they were counted by, so the last has some left).
__device__ inline int even_units(const Span& s, int n) {
  const int u = (s.units + n - 1) / n;
  return n == 1 ? u : (u + kWaves - 1) / kWaves * kWaves;
}

// The same of a cut that q8_plan_kernel left: 64 places a step.
__device__ inline Slices planned(const AttendArgs& a, int lane, int want, int b) {
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
// of sequence `b`.  Over the lanes of each wavefront alike, a sequence each.
template <int ROWS>
__device__ inline Slices cut(const Geo& g, const AttendArgs& a, int lane, int want, int b) {
#pragma clang fp contract(off)
  if (a.plan) return planned(a, lane, want, b);
  // the sums are fp32: they choose the size, alike in every wavefront and kernel, and no more
  float u = 0.0f, n = 0.0f;
  int q0, m, blocks = 0, most = 1;
  Span sp;
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

// The cut of many sequences, once for the call.  One workgroup.
template <int NB>
__global__ __launch_bounds__(1024) void q8_plan_kernel(Geo g, AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  __shared__ float units[16], segments[16];
  __shared__ int longest[16], sums[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int q0, m, blocks;
  Span sp;
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

// A workgroup of kWaves wavefronts has a slice of a segment.  target > 0: slice blockIdx.x of the
// cut; else the segment blockIdx.x = (sequence, row block, kv head) whole.
template <int HD, bool E4M3, int NB>
__global__ __launch_bounds__(64 * kWaves, decode_groups(HD, NB)) void q8_decode_kernel(Geo g,
                                                                                 AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  constexpr int LD = HD + 4;
  __shared__ __align__(16) float red[kWaves][ROWS][LD];
  __shared__ float ml[kWaves][ROWS][2];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Wave<HD, E4M3, NB> w(g, a, lane);
  Segment s;
  int u0 = 0, u1, blocks;
  bool whole = true;
  if (a.target) {
    const Slices c = cut<ROWS>(g, a, lane, blockIdx.x, 0);
    if (c.b >= a.batch) return;
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
    if (s.rb >= blocks) return;
    u1 = s.span.units;
  }
  const int left = s.m * g.gqa - s.rb * ROWS;
  s.nrows = left < ROWS ? left : ROWS;
  w.start(s);
  w.units(s, u0 + wave, u1);

  // Fold the wavefronts' parts: each leaves (m, l, acc) as they are, the reader scales.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = w.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) {
      ml[wave][nb * 16 + lane][0] = w.m[nb];
      ml[wave][nb * 16 + lane][1] = l;
    }
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
      *(f4*)&red[wave][nb * 16 + w.n16][d * 16 + w.kq * 4] = w.acc[nb][d];
  }
  __syncthreads();
  constexpr int PER = HD / 16;  // channels of a thread
  for (int i = threadIdx.x; i < s.nrows * 16; i += 64 * kWaves) {
    const int row = i / 16, ch = i % 16 * PER;
    float mm = kNegInf, l = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) mm = fmaxf(mm, ml[v][row][0]);
    float x[PER];
#pragma unroll
    for (int c = 0; c < PER; ++c) x[c] = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      // a part without a maximum saw nothing, or only NaN: l tells
      const float mv = ml[v][row][0];
      const float f = mv == kNegInf ? 1.0f : exp2_(mv - mm);
      l += ml[v][row][1] * f;
#pragma unroll
      for (int c = 0; c < PER; ++c) x[c] += red[v][row][ch + c] * f;
    }
    if (whole) {
      finish_row(g, a, s, row, HD, ch, x, PER, l, mm);
    } else {
      const int64_t at = (int64_t)blockIdx.x * a.rows + row;
#pragma unroll
      for (int c = 0; c < PER; c += 4) *(f4*)(a.part_acc + at * HD + ch + c) = *(f4*)(x + c);
      if (ch == 0) {
        a.part_ml[at * 2] = mm;
        a.part_ml[at * 2 + 1] = l;
      }
    }
  }
}

// Joins a segment's slices, in their order.  blockIdx.x: segment.  MANY: of the row blockIdx.y, the
// threads side by side share the slices; else they share the rows.
template <int HD, int NB, bool MANY>
__global__ __launch_bounds__(256) void q8_join_kernel(Geo g, AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  constexpr int TC = HD / 4;      // threads of a row
  constexpr int PG = 256 / TC;    // rows, or slices, at a time
  const int lane = threadIdx.x & 63;
  Segment s;
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
    for (int row = grp; row < s.nrows; row += PG) {
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

// Adds up the weight of every block: a lane per 16 tokens, a wavefront every fourth kv head; their
// four sums in order, then the 16s of a page.  blockIdx.y: sequence.  24 sequences of 4096 to 12289
// tokens, 40/8 heads: 5 us; with one wavefront for all kv heads 13.
template <int NB>
__global__ __launch_bounds__(256) void q8_weights_kernel(Geo g, AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  __shared__ float part[4][64];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int grp = blockIdx.x * 64 + lane;
  int q0, m, blocks;
  Span sp;
  sequence_span<ROWS>(g, a, b, &q0, &m, &sp, &blocks);
  const int t0 = grp * 16, tile = t0 / kTile;
  // groups that no unit covers were not written by this call
  const bool there = t0 < sp.n && (t0 >= sp.nq || tile < sp.ns || tile >= sp.w0);
  float sum = 0.0f;
  for (int h = __ballot(there) ? wave : g.nkv; h < g.nkv; h += 4)
    for (int rb = 0; rb < blocks; ++rb) {
      const int64_t seg = ((int64_t)b * g.nkv + h) * a.row_blocks + rb;
      const float* src = a.group_lse + (seg * a.groups + grp) * a.rows;
      const int left = m * g.gqa - rb * ROWS, rows = left < ROWS ? left : ROWS;
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const int x = rb * ROWS + r;
        const float lse = a.row_lse[(int64_t)(q0 + x / g.gqa) * g.nh + h * g.gqa + x % g.gqa];
        const float got = there ? src[r] : kNegInf;
        sum += lse == kNegInf ? 0.0f : exp2_(got - lse);
      }
    }
  part[wave][lane] = sum;
  __syncthreads();
  if (wave > 0) return;
  sum = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  const int per = g.page / 16;
  for (int d = 1; d < per; d <<= 1) sum += __shfl_xor(sum, d);
  const int page = grp / per;
  if (grp % per == 0 && page < g.max_pages) {
    float* w = a.weights + (int64_t)b * g.max_pages + page;
    *w = a.decay == 0.0f ? sum : __builtin_fmaf(a.decay, *w, sum);
  }
}

template <int HD, bool E4M3, int NB>
static void decode_kernels(const Geo& g, const AttendArgs& a, hipStream_t s) {
  const int segments = a.batch * g.nkv * a.row_blocks;
  const unsigned blocks = a.target ? a.target + segments : segments;
  if (a.plan) hipLaunchKernelGGL((q8_plan_kernel<NB>), dim3(1), dim3(1024), 0, s, g, a);
  hipLaunchKernelGGL((q8_decode_kernel<HD, E4M3, NB>), dim3(blocks), dim3(64 * kWaves), 0, s, g, a);
  if (a.target) {
    // from about 16 slices a segment on, a workgroup per row: its threads share the slices (at 8
    // to 16, 8 sequences of 100 to 3000 tokens, 16/16 heads of 64, 4 queries: 16.0 us against 14.6)
    if (a.target >= 16 * segments)
      hipLaunchKernelGGL((q8_join_kernel<HD, NB, true>), dim3(segments, a.rows), dim3(256), 0, s, g,
                         a);
    else
      hipLaunchKernelGGL((q8_join_kernel<HD, NB, false>), dim3(segments), dim3(256), 0, s, g, a);
  }
  if (a.weights)
    hipLaunchKernelGGL((q8_weights_kernel<NB>), dim3((a.groups + 63) / 64, a.batch), dim3(256), 0, s,
                       g, a);
}

// A call of no queries: max_q is 0, so no segment adds anything and the weights decay.
hipError_t launch_decay(const Geo& g, const AttendArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((q8_weights_kernel<1>), dim3((a.groups + 63) / 64, a.batch), dim3(256), 0, s, g,
                     a);
  return hipGetLastError();
}

template <int HD, bool E4M3>
static void decode_rows(const Geo& g, const AttendArgs& a, int nb, hipStream_t s) {
  if (nb == 1) decode_kernels<HD, E4M3, 1>(g, a, s);
  else decode_kernels<HD, E4M3, 2>(g, a, s);
}

hipError_t launch_decode(const Geo& g, const AttendArgs& a, int nb, hipStream_t s) {
  const bool e = g.codes == JACQ_Q8_E4M3;
  if (g.hd == 128) {
    if (e) decode_rows<128, true>(g, a, nb, s);
    else decode_rows<128, false>(g, a, nb, s);
  } else {
    if (e) decode_rows<64, true>(g, a, nb, s);
    else decode_rows<64, false>(g, a, nb, s);
  }
  return hipGetLastError();
}

}  // namespace q8
}  // namespace jacq
