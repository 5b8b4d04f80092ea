// kivi_few.hip -- attention of a few queries per sequence over the int4 cache.
//
// A segment is a (sequence, kv head, block of 16 NB query rows); a row is a (query token, head of the
// kv head's group), so all G heads share every byte.  Its units of 32 tokens are dealt to the 4
// wavefronts of a workgroup, or of several, whose parts a second kernel joins.  Per unit and wavefront:
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16.  The tokens that a K operand's rows are
// (tok_k) are such that a lane's P is already its next operand (tok_v); a lane's V operands are 8 of its
// own tokens by 8 (HD 64: 4) of its own channels, so a dword of codes a token serves all of them.
//   K[t, d] = code s_d + z_d (of the group),  V[t, d] = code s_t + z_t (of 32 channels)
// are rounded to fp16 once, for the matrix cores; sums, maxima and weights are fp32.
//
// A group's codes, scales and zeros (40 HD bytes) come by LDS DMA, a ring of units ahead.
//
// Bound by issue, not by memory: of HD 128 a unit is about 380 vector instructions for 32 rows, 320
// for 16 (200 of them codes to fp16, which every row shares), for 5 KB.  32 sequences of 1500 to 6007 tokens, 40/8 heads
// of 128, 4 queries: 53 us where the bytes alone take 35; 64 of 1024 to 16384 under a window of 4096, 32/8
// heads, one query: 70 us, as long as the bytes.  A sliced call has 13 us of its own: two launches, the cut,
// the join.
#include "kivi_attend.h"
#include "kivi_stage.h"

namespace jacq {

namespace {

template <int HD>
struct FewStage {
  uint8_t k[32 * HD / 2];
  uint8_t v[32 * HD / 2];
  uint8_t s[8 * HD];  // scale and zero of K [HD], then of V [32][HD / 32]
};

// Stages of a wavefront's ring, by what the LDS holds for few_groups workgroups (5 KB a stage of HD 128).
template <int HD, int NB>
constexpr int few_stages() { return HD == 64 ? 4 : NB == 1 ? 2 : 3; }

__device__ inline int table_at(const int32_t* row, int i) {  // uniform: a scalar load
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(row + i);
}

template <int HD, int P, int NB>
struct Few {
  static constexpr int KS = HD / 32;   // k-steps of S^T
  static constexpr int CPL = HD / 16;  // channels of a lane's V: operands of O^T
  static constexpr int S = few_stages<HD, NB>();
  typedef typename Cfg<HD, P>::kvec kvec;
  const KiviGeo& g;
  const KiviAttendArgs& a;
  int lane, n16, kq;

  h8 q[NB][KS];
  float qs[NB];  // a row's scores are qs times what the matrix cores give (log2(e) included)
  int pos[NB];   // the last token that the row sees
  f4 acc[NB][CPL];
  float m[NB], l[NB];

  __device__ Few(const KiviGeo& g_, const KiviAttendArgs& a_, int lane_)
      : g(g_), a(a_), lane(lane_), n16(lane_ & 15), kq(lane_ >> 4) {}

  __device__ int position(const Segment<KiviGeo>& s, int row) const {
    return a.causal ? s.span.first + row / g.gqa : s.span.n - 1;
  }

  __device__ void start(const Segment<KiviGeo>& s) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = s.rb * 16 * NB + nb * 16 + n16;
      const int tok = row / g.gqa, head = s.h * g.gqa + row % g.gqa;
      const bool ok = tok < s.m;
      pos[nb] = ok ? position(s, row) : -1;
      m[nb] = kNegInf;
      l[nb] = 0.0f;
#pragma unroll
      for (int j = 0; j < CPL; ++j) acc[nb][j] = f4{0, 0, 0, 0};
      const uint16_t* src =
          a.q + (int64_t)(s.q0 + (ok ? tok : 0)) * a.q_stride + head * HD + kq * (HD / 4);
      u4 raw[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) raw[i] = ok ? *(const u4*)(src + 8 * i) : u4{0, 0, 0, 0};
      qs[nb] = half_row(raw, a.q_bf16, a.scale, q[nb], [](float x) {
        x = fmaxf(x, __shfl_xor(x, 16));
        return fmaxf(x, __shfl_xor(x, 32));
      });
    }
  }

  // Whether some rows of the block do not see all of a unit.
  struct Seen {
    int first, last;  // positions of the block's first and last row
    __device__ bool part(const KiviAttendArgs& a, int t0) const {
      return t0 + kGroup - 1 > first ||
             (a.window > 0 && t0 <= last - a.window && t0 + kGroup > a.sinks);
    }
  };

  // Both products of a unit.  This lane's 8 tokens are tok_v(kq, e) of the unit at t0; those of `poison`
  // are NaN to the rows that see them.  All row blocks side by side, under one branch: their chains of
  // dependent instructions fill each other's waits.  v(odd, x): the V operands of the even or odd
  // channels of this lane, made when they are needed: registers are what limits the wavefronts a SIMD.
  template <class V>
  __device__ void unit(const h8 (&k)[2][KS], int t0, bool masked, bool weeds, uint32_t poison, V v) {
    f4 sc[NB][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          sc[nb][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[tt][i], q[nb][i],
                                                              i ? sc[nb][tt] : f4{0, 0, 0, 0}, 0, 0, 0);
    if (weeds) {  // uniform, as masked is
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sc[nb][e / 4][e & 3] = poison >> e & 1 ? __builtin_nanf("") : sc[nb][e / 4][e & 3];
    }
    if (masked) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sc[nb][e / 4][e & 3] = sees(t0 + tok_v(kq, e), pos[nb], a.window, a.sinks)
                                     ? sc[nb][e / 4][e & 3] : kNegInf;
    }
    float mx[NB];
    bool grows = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const f4 x = sc[nb][0], y = sc[nb][1];
      mx[nb] = max3f(max3f(x.x, x.y, x.z), max3f(x.w, y.x, y.y), max2f(y.z, y.w));
      mx[nb] = max_xor32(max_xor16(mx[nb])) * qs[nb];
      grows = grows || mx[nb] > m[nb] + (kLift + kSlack);
    }
    if (__ballot(grows)) {  // also where m is -inf and mx is not
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float to = mx[nb] > m[nb] + (kLift + kSlack) ? mx[nb] - kLift : m[nb];
        const float f = to > m[nb] ? exp2_(m[nb] - to) : 1.0f;
        m[nb] = to;
        l[nb] *= f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) acc[nb][j] *= f;
      }
    }
    h8 p[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float base = m[nb] == kNegInf ? 0.0f : -m[nb];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = exp2_(__builtin_fmaf(sc[nb][e / 4][e & 3], qs[nb], base));
        l[nb] += w;
        p[nb][e] = (_Float16)w;
      }
    }
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      h8 x[CPL / 2];
      v(odd, x);
#pragma unroll
      for (int c = 0; c < CPL / 2; ++c)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          acc[nb][2 * c + odd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[c], p[nb], acc[nb][2 * c + odd], 0,
                                                                        0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // An int4 group in the LDS.  gone: bit i: its tokens 16 i on lie in a page outside the pool.
  __device__ void group(const FewStage<HD>* st, int t0, bool masked, int gone) {
    h8 k[2][KS];
    {
      kvec code[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        code[tt] = *(const kvec*)(st->k + tok_k(tt, n16) * (HD / 2) + kq * (HD / 8));
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const u4 s = *(const u4*)(st->s + kq * (HD / 2) + 16 * i);
        const u4 z = *(const u4*)(st->s + 2 * HD + kq * (HD / 2) + 16 * i);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) k[tt][i] = values8(code[tt][i], s, z);
      }
    }
    // All scales and zeros of V, a few a lane: below 4096, 15 scale + |zero| is a finite fp16.
    typedef uint32_t few_t __attribute__((ext_vector_type(HD / 64)));
    const few_t some = *(const few_t*)(st->s + 4 * HD + lane * (HD / 16));
    const uint32_t most = most_bits(some[0], some[HD / 64 - 1]);
    // scales and zeros of this lane's 8 tokens, two by two
    const uint8_t* at = st->s + 4 * HD + 2 * (tok_v(kq, 0) * (HD / 32) + n16 * CPL / 32);
    constexpr int STEP = 2 * 2 * (HD / 32);  // two tokens on
    uint32_t s[4], z[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      s[p] = *(const uint16_t*)(at + 2 * p * STEP) | (uint32_t)*(const uint16_t*)(at + (2 * p + 1) * STEP) << 16;
      z[p] = *(const uint16_t*)(at + 2 * HD + 2 * p * STEP) |
             (uint32_t)*(const uint16_t*)(at + 2 * HD + (2 * p + 1) * STEP) << 16;
    }
    uint32_t poison = 0;
    const bool weeds = gone || __ballot(either_half(most) >= 0x6c00u);
    if (weeds) poison = weed(s, z, gone);
    const uint8_t* vc = st->v + tok_v(kq, 0) * (HD / 2) + n16 * (CPL / 2);
    typedef typename std::conditional<HD == 128, uint32_t, uint16_t>::type code_t;
    code_t code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = *(const code_t*)(vc + e * HD);
    unit(k, t0, masked, weeds, poison, [&](int odd, h8 (&x)[CPL / 2]) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        h2 y[CPL / 2];
        if constexpr (HD == 128) values8x2(code[2 * p], code[2 * p + 1], odd, pair(s[p]), pair(z[p]), y);
        else values4x2(code[2 * p] | (uint32_t)code[2 * p + 1] << 16, odd, pair(s[p]), pair(z[p]), y);
#pragma unroll
        for (int c = 0; c < CPL / 2; ++c) {
          x[c][2 * p] = y[c].x;
          x[c][2 * p + 1] = y[c].y;
        }
      }
    });
  }

  // A token's V that is not finite, or not there, must reach no row that does not see it, and a
  // weight of 0 would not keep it out: it becomes 0 (s and z of this lane's tokens), and its key NaN,
  // which the mask keeps out.  Returns the bits of this lane's tokens.
  __device__ uint32_t weed(uint32_t (&s)[4], uint32_t (&z)[4], int gone) const {
    uint32_t bad = gone >> (kq >> 1) & 1 ? 255u : 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float sc = h2f_((uint16_t)(s[e / 2] >> 16 * (e & 1))), ze = h2f_((uint16_t)(z[e / 2] >> 16 * (e & 1)));
      if (!holds(sc, ze)) bad |= 1u << e;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t keep = (bad >> 2 * p & 1 ? 0u : 0xffffu) | (bad >> (2 * p + 1) & 1 ? 0u : 0xffff0000u);
      s[p] &= keep;
      z[p] &= keep;
    }
    return any16(bad);
  }
  // The bits of the 16 lanes that have this lane's tokens.
  __device__ static uint32_t any16(uint32_t bad) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) bad |= __shfl_xor(bad, d);
    return bad;
  }

  // 32 fp16 tokens from t0 on, at most; what lies behind the last one is not read: the last one stands
  // for it, and no row sees it.
  __device__ void recent(const Segment<KiviGeo>& s, int t0, bool masked) {
    const int64_t base = (((int64_t)s.b * g.nkv + s.h) * g.rs + (t0 - s.span.old)) * HD;
    const int last = s.span.n - t0 - 1;
    const uint16_t *ks = a.pool.k_scr + base, *vs = a.pool.v_scr + base;
    h8 k[2][KS];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int r = tok_k(tt, n16);
      const uint32_t at = (r < last ? r : last) * HD + kq * (HD / 4);
#pragma unroll
      for (int i = 0; i < KS; ++i) k[tt][i] = *(const h8*)(ks + at + 8 * i);
    }
    typedef uint32_t row_t __attribute__((ext_vector_type(CPL / 2)));
    row_t x[8];
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = tok_v(kq, e);
      x[e] = *(const row_t*)(vs + (uint32_t)((r < last ? r : last) * HD + n16 * CPL));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int c = 0; c < CPL / 2; ++c) most = most_bits(most, x[e][c]);
    uint32_t poison = 0;
    const bool weeds = __ballot(either_half(most) >= 0x7c00u);
    if (weeds) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t mine = 0;
#pragma unroll
        for (int c = 0; c < CPL / 2; ++c) mine = most_bits(mine, x[e][c]);
        if (either_half(mine) >= 0x7c00u) {
          poison |= 1u << e;
          x[e] = row_t(0);
        }
      }
      poison = any16(poison);
    }
    unit(k, t0, masked, weeds, poison, [&](int odd, h8 (&v)[CPL / 2]) {
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int c = 0; c < CPL / 2; ++c) {
          const h2 y = pair(__builtin_amdgcn_perm(x[2 * p + 1][c], x[2 * p][c],
                                                  odd ? 0x07060302u : 0x05040100u));
          v[c][2 * p] = y.x;
          v[c][2 * p + 1] = y.y;
        }
    });
  }

  // Units u0, u0 + kSliceWaves, ... below u1, but those of which no row of this block sees anything:
  // behind the last row, and between the sinks and the first row's window.
  __device__ void units(const Segment<KiviGeo>& s, FewStage<HD>* ring, int u0, int u1) {
    const KiviSpan& sp = s.span;
    Seen seen;
    seen.first = uniform(position(s, s.rb * 16 * NB));
    seen.last = uniform(position(s, s.rb * 16 * NB + s.nrows - 1));
    // the units of this block's window, [lo, hi)
    const int hi = seen.last < 0 ? 0 : sp.ns + (seen.last / kGroup + 1 - sp.w0);
    int lo = sp.ns;
    if (a.window > 0 && seen.first >= a.window)
      lo = sp.ns + ((seen.first - a.window + 1) / kGroup - sp.w0);
    u1 = u1 < hi ? u1 : hi;
    const int sinks = a.window > 0 ? (int)(((int64_t)a.sinks + kGroup - 1) / kGroup) : 0;  // units of them
    auto next = [&](int u) {  // u, or behind what lies between the sinks and lo
      return u >= sinks && u < lo ? u + (lo - u + kSliceWaves - 1) / kSliceWaves * kSliceWaves : u;
    };
    const StageBases sb = stage_bases<HD, P>(a.pool, g.nkv, s.h, lane);
    const int32_t* table = a.tables + (int64_t)s.b * g.max_pages;
    int at = next(u0), ahead = at, p0 = 0, p1 = 0;
    auto look = [&] {  // the pages of unit `ahead`, if it is a group
      if (ahead >= u1) return;
      const int t = sp.tile_of(ahead);
      if (t * kGroup >= sp.old) {
        ahead = u1;  // fp16 from here on
        return;
      }
      p0 = table_at(table, P == 16 ? 2 * t : t);
      p1 = P == 16 ? table_at(table, 2 * t + 1) : p0;
    };
    int put = 0, get = 0, flying = 0;
    uint32_t gone = 0;  // two bits for each unit in flight
    auto issue = [&] {
      const bool no0 = (uint32_t)p0 >= (uint32_t)g.num_pages, no1 = (uint32_t)p1 >= (uint32_t)g.num_pages;
      // nothing still reads the stage
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      load_stage<HD, P>(ring + put, sb, no0 ? 0 : p0, no1 ? 0 : p1, lane);
      // a group's scales of K are in its first page
      gone |= ((no0 ? 3u : 0u) | (no1 ? 2u : 0u)) << 2 * flying;
      put = put + 1 == S ? 0 : put + 1;
      ++flying;
      ahead = next(ahead + kSliceWaves);
      look();
    };
    look();
    constexpr int L = stage_loads<HD>();
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (ahead < u1) issue();
    while (flying) {
      if (ahead < u1) issue();
      if (S >= 4 && flying >= 4) wait_vm<3 * L>();
      else if (S >= 3 && flying >= 3) wait_vm<2 * L>();
      else if (flying >= 2) wait_vm<L>();
      else wait_vm<0>();
      const int t0 = sp.tile_of(at) * kGroup;
      group(ring + get, t0, seen.part(a, t0), (int)(gone & 3u));
      gone >>= 2;
      get = get + 1 == S ? 0 : get + 1;
      --flying;
      at = next(at + kSliceWaves);
    }
    for (; at < u1; at = next(at + kSliceWaves)) {
      const int t0 = sp.tile_of(at) * kGroup;
      recent(s, t0, seen.part(a, t0));
    }
  }
};

}  // namespace

// Units of a slice, from the call's units, its segments and the longest one's units.  Segments stay whole
// if none is much longer than a CU's share and they fill the CUs evenly: 32 of 1900 to 2100 tokens, 6
// queries, 40/8 heads of 128, whole 34.6 us, cut 35.8; but 8 of 1000 to 4000, a query of 32/32 heads, 46 and
// 32.  Else slices are a CU's share, so that few of them are joined, but 8 units at least (less is all
// fixed cost) and 32 at most (16 us of a wavefront: the tail), and no more than there is room for.
__device__ inline int slice_units(const KiviAttendArgs& a, float all, float segments, int longest) {
#pragma clang fp contract(off)  // the kernel and its join have to find the same size
  const float cus = (float)a.cus;
  const bool even = a.rows > 16 || segments >= 0.8f * cus * __builtin_ceilf(segments / cus);
  if ((float)longest <= 1.2f * all / cus + 8.0f &&
      (segments <= cus || (even && all >= 0.75f * segments * (float)longest)))
    return longest;
  const int fair = (int)(all / cus) + 1;  // one slice a CU
  const int few = fair < 8 ? 8 : fair > 32 ? 32 : fair;
  const float fit = (float)a.target - 0.5f * segments, half = 0.5f * (float)a.target;
  const int many = (int)(all / (fit > half ? fit : half)) + 1;
  return ((many > few ? many : few) + kSliceWaves - 1) / kSliceWaves * kSliceWaves;
}

template <int HD, int P, int NB>
__global__ __launch_bounds__(64 * kSliceWaves, few_groups(HD, NB)) void kivi_few_kernel(
    KiviGeo g, KiviAttendArgs a) {
  constexpr int LD = HD + 4, S = few_stages<HD, NB>();
  struct Parts {
    float red[kSliceWaves][16][LD];
    float ml[kSliceWaves][16][2];
  };
  constexpr size_t RING = sizeof(FewStage<HD>) * S * kSliceWaves;
  __shared__ __align__(16) uint8_t shared[RING > sizeof(Parts) ? RING : sizeof(Parts)];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Segment<KiviGeo> s;
  int u0, u1;
  bool whole;
  if (!place_slice<16 * NB>(g, a, lane, s, u0, u1, whole)) return;
  Few<HD, P, NB> w(g, a, lane);
  w.start(s);
  w.units(s, (FewStage<HD>*)shared + wave * S, uniform(u0 + wave), uniform(u1));

  // Fold the wavefronts' parts, which take the rings' place: 16 rows at a time.
  Parts& parts = *(Parts*)shared;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    __syncthreads();
    float l = w.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) {
      parts.ml[wave][lane][0] = w.m[nb];
      parts.ml[wave][lane][1] = l;
    }
    // O^T row 4 kq + r of operand j is channel CPL (4 kq + r) + j
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < HD / 16; j += 4)
        *(f4*)&parts.red[wave][w.n16][(4 * w.kq + r) * (HD / 16) + j] =
            f4{w.acc[nb][j][r], w.acc[nb][j + 1][r], w.acc[nb][j + 2][r], w.acc[nb][j + 3][r]};
    __syncthreads();
    const int left = s.nrows - 16 * nb;
    fold_parts<HD>(g, a, s, whole, parts.red, parts.ml, 16 * nb, left < 16 ? left : 16);
  }
}

template <int NB>
__global__ __launch_bounds__(1024) void kivi_few_plan_kernel(KiviGeo g, KiviAttendArgs a) {
  plan_cut<16 * NB>(g, a);
}

template <int HD, int NB, bool MANY>
__global__ __launch_bounds__(256) void kivi_few_join_kernel(KiviGeo g, KiviAttendArgs a) {
  join_slices<HD, 16 * NB, MANY>(g, a);
}

template <int HD, int P, int NB>
static hipError_t few_kernels(const KiviGeo& g, const KiviAttendArgs& a, hipStream_t s) {
  const int segments = a.batch * g.nkv * a.row_blocks;
  const unsigned blocks = a.target ? a.target + segments : segments;
  if (a.plan) hipLaunchKernelGGL((kivi_few_plan_kernel<NB>), dim3(1), dim3(1024), 0, s, g, a);
  hipLaunchKernelGGL((kivi_few_kernel<HD, P, NB>), dim3(blocks), dim3(64 * kSliceWaves), 0, s, g, a);
  if (a.target) {
    if (a.target >= 16 * segments)
      hipLaunchKernelGGL((kivi_few_join_kernel<HD, NB, true>), dim3(segments, a.rows), dim3(256), 0, s,
                         g, a);
    else
      hipLaunchKernelGGL((kivi_few_join_kernel<HD, NB, false>),
                         dim3(segments, (a.rows * HD + 1023) / 1024), dim3(256), 0, s, g, a);
  }
  return hipGetLastError();
}

template <int HD, int P>
static hipError_t few_rows(const KiviGeo& g, const KiviAttendArgs& a, int nb, hipStream_t s) {
  return nb == 1 ? few_kernels<HD, P, 1>(g, a, s) : few_kernels<HD, P, 2>(g, a, s);
}

hipError_t launch_attend_few(const KiviGeo& g, const KiviAttendArgs& a, int nb, hipStream_t s) {
  if (g.hd == 128) return g.page == 16 ? few_rows<128, 16>(g, a, nb, s) : few_rows<128, 32>(g, a, nb, s);
  return g.page == 16 ? few_rows<64, 16>(g, a, nb, s) : few_rows<64, 32>(g, a, nb, s);
}

}  // namespace jacq
