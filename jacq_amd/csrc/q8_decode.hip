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

  __device__ void start(const Segment<Geo>& s) {
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
  __device__ int page_of(const Segment<Geo>& s, int t) const {
    const int last = s.span.nq - 16;  // never past the sequence's own entries
    t = t < last ? t : last;
    return a.tables[(int64_t)s.b * g.max_pages + (t >> g.page_log2)];
  }
  __device__ bool exists(int page) const { return page >= 0 && page < g.num_pages; }
  __device__ uint32_t held(int page) const { return exists(page) ? page : 0; }

  __device__ void pages(const Segment<Geo>& s, int tile, int& pk, int& pv) const {
    pk = page_of(s, tile * kTile + n16 / 4 * 16);
    pv = page_of(s, tile * kTile + kq * 16);
  }

  // A quantised tile's K codes, its scales and its V codes.  A tile begins a page or lies in one, so
  // where a lane reads in its page is the same for all.
  __device__ void load_k(const Segment<Geo>& s, int pk, Codes& c) const {
    uint32_t in = (s.h * g.page + (n16 / 4 * 16 & (g.page - 1)) + (n16 & 3)) * HD + kq * 16;
    asm volatile("" : "+v"(in));  // one register over the loop, not a pointer's two
    const uint8_t* k = a.pool.k_code + ((uint64_t)held(pk) * (uint32_t)(g.nkv * g.page * HD) + in);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < KL; ++j) c.k[t][j] = *(const u4*)(k + t * 4 * HD + j * 64);
  }
  __device__ void load_scales(const Segment<Geo>& s, int pv, Codes& c) const {
    const uint64_t slot = (uint64_t)held(pv) * (uint32_t)g.nkv + (uint32_t)s.h;
    c.ks = a.pool.k_scale[slot];
    c.there = exists(pv);
    c.vs = a.pool.v_scale[slot];
  }
  __device__ void load_v(const Segment<Geo>& s, int pv, Codes& c) const {
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
  __device__ void store_group(const Segment<Geo>& s, int t0, int end) const {
    if (!a.weights || t0 >= end) return;
    const int64_t seg = ((int64_t)s.b * g.nkv + s.h) * a.row_blocks + s.rb;
    float* dst = a.group_lse + (seg * a.groups + (t0 >> 4)) * a.rows;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (nb * 16 + n16 < s.nrows) dst[nb * 16 + n16] = group[nb];
  }

  __device__ bool needs_mask(const Segment<Geo>& s, int t0, int end) const {
    // uniform: the tile's 64 tokens are all there and every row sees them
    const int first = s.span.first + s.rb * 16 * NB / g.gqa;
    const int last = s.span.first + (s.rb * 16 * NB + s.nrows - 1) / g.gqa;
    return t0 + kTile > end || t0 + kTile - 1 > first ||
           (a.window > 0 && t0 <= last - a.window && t0 + kTile > a.sinks);
  }

  // No row sees the 16 tokens from t on, as their windows begin later: their page may be any, and
  // its e4m3 codes NaN, which a weight of 0 would not take out.
  __device__ bool before_window(const Segment<Geo>& s, int t) const {
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
  __device__ void tail(const Segment<Geo>& s) {
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

  // Units u0, u0 + kSliceWaves, ... below u1.  One set of code registers: the next tile's K is
  // loaded when this one's scores are done, its V when this one's is used up.
  __device__ void units(const Segment<Geo>& s, int u0, int u1) {
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
      if (u0 + kSliceWaves < e) pages(s, sp.tile_of(u0 + kSliceWaves), nk, nv);
      for (;;) {
        const int next = u0 + kSliceWaves < e ? sp.tile_of(u0 + kSliceWaves) : -1;
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
        u0 += kSliceWaves;
        if (next < 0) break;
        load_scales(s, nv, c);
        load_v(s, nv, c);
        // behind the loads: what is loaded behind a store waits for it too (256 sequences of 100 to
        // 4000 tokens, 32/8 heads of 128: 241 us against 246)
        store_group(s, t0 + kq * 16, sp.nq);
        if (u0 + kSliceWaves < e) pages(s, sp.tile_of(u0 + kSliceWaves), nk, nv);
        tile = next;
      }
      store_group(s, tile * kTile + kq * 16, sp.nq);
    }
    if (u0 < u1) tail(s);  // the unit behind the quantised ones
  }
};

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
  return ((many > few ? many : few) + kSliceWaves - 1) / kSliceWaves * kSliceWaves;
}

template <int NB>
__global__ __launch_bounds__(1024) void q8_plan_kernel(Geo g, AttendArgs a) {
  plan_cut<16 * NB>(g, a);
}

// A workgroup of kSliceWaves wavefronts has a slice of a segment.  target > 0: slice blockIdx.x of the
// cut; else the segment blockIdx.x = (sequence, row block, kv head) whole.
template <int HD, bool E4M3, int NB>
__global__ __launch_bounds__(64 * kSliceWaves, decode_groups(HD, NB)) void q8_decode_kernel(Geo g,
                                                                                 AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  constexpr int LD = HD + 4;
  __shared__ __align__(16) float red[kSliceWaves][ROWS][LD];
  __shared__ float ml[kSliceWaves][ROWS][2];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Wave<HD, E4M3, NB> w(g, a, lane);
  Segment<Geo> s;
  int u0, u1;
  bool whole;
  if (!place_slice<ROWS>(g, a, lane, s, u0, u1, whole)) return;
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
  fold_parts<HD>(g, a, s, whole, red, ml, 0, s.nrows);
}

template <int HD, int NB, bool MANY>
__global__ __launch_bounds__(256) void q8_join_kernel(Geo g, AttendArgs a) {
  join_slices<HD, 16 * NB, MANY>(g, a);
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
  hipLaunchKernelGGL((q8_decode_kernel<HD, E4M3, NB>), dim3(blocks), dim3(64 * kSliceWaves), 0, s, g, a);
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
