// q8_prefill.hip -- attention of prompts over the 8-bit cache.
//
// A workgroup has 128 query rows of one kv head (row = query token x head of
// the group), 32 for each of 4 wavefronts, and goes through the tiles of 64
// tokens that any of its rows sees, or through one of several slices of them.
// A tile's codes are converted to fp16 once and shared through the LDS.
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_f16; a lane's column is
// a query row, so its maximum, sum and rescaling are the lane's own (and its
// partner's, 32 lanes on), and the order in which K's rows enter makes P the
// next operand as it stands.  The scales of 16 tokens are the wavefront's:
// t = s (ks q) + log2(vs), as in q8_decode.hip, where the reason is.
//
// Bound by the matrix cores, the LDS and the vector units taking turns.  A prompt of
// 8191 tokens (40/8 heads of 128, int8): 780 to 820 us, 840 to 880 TFLOP/s, where
// the library's product of 8192^3 runs at 1145 to 1242.  Of the CUs' cycles the matrix
// cores are busy for 40 %, the vector units for 56 %, the LDS for 53 %.  Without the
// staging it takes 586 us, without the softmax 629, the products with their
// LDS reads alone 526: an operand feeds one product, since 64 rows a wavefront
// (two products each) do not fit the registers at HD 128 (spills, 1061 us).
// On zeros the same prompt takes 702 us against 854 on random values (one card), the
// matrix instructions alone 310 and 435: what they do not account for, about 400 us,
// is the other work that does not run beside them.
// Two workgroups a CU, not in step: one's products run beside the other's
// softmax.  The softmax of a half tile among the next half's products, in one
// wavefront's order, was as fast (HD 128: 820 us; HD 64: 204 against 213).
#include <type_traits>

#include "q8_common.h"

namespace jacq {
namespace q8 {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = kPrefillRows;
static_assert(kRows == 32 * kWaves, "32 a wavefront");
constexpr float kNegInf = -__builtin_inff();

template <int HD>
struct Lds {
  uint16_t k[2][kTile][HD];    // 16-byte chunks of a row are XOR-ed with the row
  uint16_t v[2][HD][kTile];
  float ks[4][4], lvs[4][4], ivs[4][4];  // per 16 tokens: K scale, log2 and inverse of V's
};

// LDS writes are done, loads from memory may be in flight.
__device__ inline void turn() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Where chunk c (8 values) of a row lies, so that 16 rows' same chunk covers all banks.
template <int HD>
__device__ inline int k_chunk(int row, int c) {
  return HD == 128 ? c ^ (row & 15) : c ^ (row >> 1 & 7);
}
__device__ inline int v_chunk(int d, int c) { return c ^ (d >> 1 & 7); }

// The value of the lane 32 on (or back).
__device__ inline float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}

// 4 values of O, in its type.
__device__ inline void store4(const AttendArgs& a, int64_t at, f4 x) {
  if (a.o_type == JACQ_Q8_FP32) {
    *(f4*)((float*)a.o + at) = x;
    return;
  }
  const bool bf = a.o_type == JACQ_Q8_BF16;
  const uint32_t x0 = bf ? f2bf(x.x) : f2h_(x.x), x1 = bf ? f2bf(x.y) : f2h_(x.y);
  const uint32_t x2 = bf ? f2bf(x.z) : f2h_(x.z), x3 = bf ? f2bf(x.w) : f2h_(x.w);
  *(u2*)((uint16_t*)a.o + at) = u2{x0 | x1 << 16, x2 | x3 << 16};
}

// Bits 0 to n - 1; n in any range.
__device__ inline uint64_t low_bits(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << n) - 1;
}

template <int HD, bool E4M3>
__global__ __launch_bounds__(kThreads, 2) void q8_prefill_kernel(Geo g, AttendArgs a) {
  constexpr int KS = HD / 16;                        // k-steps of S^T
  constexpr int DT = HD / 32;                        // channel tiles
  constexpr int KC = kTile * HD / 16 / kThreads;     // 16-code chunks of K (and of V) a thread stages
  extern __shared__ __align__(16) uint8_t shared_bytes[];
  Lds<HD>& lds = *(Lds<HD>*)shared_bytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int h = blockIdx.x % g.nkv, slice = blockIdx.y;
  const Place place = place_of(g, a, blockIdx.x / g.nkv, g.gqa, kRowsLog2);
  const int b = place.b, q0 = place.q0, n = place.n;
  const int rows = place.m * g.gqa;
  const int rt = (rows + kRows - 1) / kRows - 1 - place.at;  // the longest first
  if (rt < 0 || place.at < 0) return;
  const int slices = uniform(prefill_slices(a, n));
  if (slice >= slices) return;
  // positions: the first query's, then the workgroup's and the wavefront's rows
  const int p0 = n - place.all;
  const int end_row = rows < (rt + 1) * kRows ? rows : (rt + 1) * kRows;
  const int pfirst = uniform(p0 + rt * kRows / g.gqa);
  const int plast = uniform(p0 + (end_row - 1) / g.gqa);
  const int wr0 = rt * kRows + wave * 32;
  const int wr1 = wr0 + 32 < rows ? wr0 + 32 : rows;
  const int wfirst = uniform(p0 + wr0 / g.gqa);
  const int wlast = uniform(wr0 < rows ? p0 + (wr1 - 1) / g.gqa : -1);

  const int row = wr0 + n32;
  const bool ok = row < rows;
  const int tok = ok ? row / g.gqa : 0, head = h * g.gqa + row % g.gqa;
  const int pos = ok ? p0 + tok : -1;
  h8 q[KS];
  float qs = a.scale, mx = kNegInf, l = 0.0f;
  f16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f16v{};
  {
    const uint16_t* src = a.q + (int64_t)(q0 + tok) * a.q_stride + head * HD + hh * 8;
    u4 raw[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) raw[i] = ok ? *(const u4*)(src + i * 16) : u4{0, 0, 0, 0};
    if (a.q_bf16) {  // as in q8_decode.hip: a power of two per row takes bf16 into fp16's range
      float big = 0.0f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c)
          big = fmaxf(big, __builtin_fabsf(__uint_as_float(c & 1 ? raw[i][c / 2] & 0xffff0000u
                                                                 : raw[i][c / 2] << 16)));
      big = fmaxf(big, other_half(big));
      const bool plain = !(big > 0.0f && big < __builtin_inff());
      const int e = plain ? 0 : 14 - __builtin_amdgcn_frexp_expf(big);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c)
          q[i][c] = (_Float16)__builtin_amdgcn_ldexpf(
              __uint_as_float(c & 1 ? raw[i][c / 2] & 0xffff0000u : raw[i][c / 2] << 16), e);
      qs = __builtin_amdgcn_ldexpf(a.scale, -e);
    } else {
#pragma unroll
      for (int i = 0; i < KS; ++i) q[i] = __builtin_bit_cast(h8, raw[i]);
    }
  }

  // Tiles: the sinks', the window's up to the last row's position; of them this slice's, from
  // `from` on.  Then the tail, the last slice's.
  const Span sp(g, n, pfirst, a.window, a.sinks);
  int top = plast < 0 ? 0 : (plast >> 6) + 1;
  top = top > sp.tiles ? sp.tiles : top;
  const int every = plast < 0 ? 0 : sp.ns + (top > sp.w0 ? top - sp.w0 : 0);
  const int from = uniform((int)((int64_t)every * slice / slices));
  const int quant = uniform((int)((int64_t)every * (slice + 1) / slices)) - from;

  // ---- staging: a thread has KC chunks of K and of V ----
  // K chunk i: 16 codes (kcc) of row kr + i 64 / KC.  V chunk i: 16 tokens (group vg) of channel
  // vd; those of a page side by side in memory.  A wavefront's chunks are 8 or 16 rows of K, and
  // at most a page of V: one page each, so the table is read once per wavefront.
  const int per = g.page >> 4, per_log2 = g.page_log2 - 4;
  const int kr = tid / (HD / 16), kcc = tid % (HD / 16);
  constexpr int KR = kTile / KC;
  uint32_t k_off[KC], v_off[KC];
  int kt[KC], vt[KC], ks0[KC], ks1[KC], vs0[KC], vs1[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int r = kr + i * KR;
    k_off[i] = (h * g.page + (r & (g.page - 1))) * HD + kcc * 16;
    kt[i] = uniform(r & -16);
    ks0[i] = r * HD + k_chunk<HD>(r, 2 * kcc) * 8;
    ks1[i] = r * HD + k_chunk<HD>(r, 2 * kcc + 1) * 8;
    const int chunk = tid + i * kThreads, in = chunk & (HD * per - 1), vd = in >> per_log2;
    const int vg = (chunk / HD >> per_log2 << per_log2) + (in & (per - 1));
    v_off[i] = (h * HD + vd) * g.page + ((vg * 16) & (g.page - 1));
    vt[i] = uniform(vg * 16 & -g.page);
    vs0[i] = vd * kTile + v_chunk(vd, 2 * vg) * 8;
    vs1[i] = vd * kTile + v_chunk(vd, 2 * vg + 1) * 8;
  }
  const int64_t stride = (int64_t)g.nkv * g.page * HD;
  const int32_t* table = a.tables + (int64_t)b * g.max_pages;
  // Units past the last one are fetched as the last one again, and never used: the loop's loads
  // have no branches around them, so each is waited for by itself, a unit after its issue.
  auto tile_at = [&](int u) { return sp.tile_of(from + (u < quant ? u : quant - 1)) * kTile; };
  auto page_at = [&](int t) {
    const int last = sp.nq - 16;
    return table[(t < last ? t : last) >> g.page_log2];
  };
  auto exists = [&](int page) { return page >= 0 && page < g.num_pages; };
  u4 kc[KC], vc[KC];
  float scale_k = 0, scale_v = 0;
  bool no_page = false, no_v[KC];
  int pk[KC], pv[KC], ps = 0;
  auto pages_k = [&](int u) {
    const int t0 = tile_at(u);
#pragma unroll
    for (int i = 0; i < KC; ++i) pk[i] = page_at(t0 + kt[i]);
    if (wave == 0) ps = page_at(t0 + (lane & 3) * 16);
  };
  auto pages_v = [&](int u) {
    const int t0 = tile_at(u);
#pragma unroll
    for (int i = 0; i < KC; ++i) pv[i] = page_at(t0 + vt[i]);
  };
  auto fetch_k = [&] {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int page = uniform(pk[i]);
      kc[i] = *(const u4*)(a.pool.k_code + (exists(page) ? page : 0) * stride + k_off[i]);
    }
    if (wave == 0) {
      const int64_t s = (int64_t)(exists(ps) ? ps : 0) * g.nkv + h;
      scale_k = a.pool.k_scale[s];
      scale_v = a.pool.v_scale[s];
      no_page = !exists(ps);
    }
  };
  auto fetch_v = [&] {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int page = uniform(pv[i]);
      no_v[i] = !exists(page);
      vc[i] = *(const u4*)(a.pool.v_code + (exists(page) ? page : 0) * stride + v_off[i]);
    }
  };
  auto stage_k = [&](int u) {
    uint16_t* dst = &lds.k[u & 1][0][0];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      *(h8*)(dst + ks0[i]) = codes8<E4M3>(kc[i].x, kc[i].y);
      *(h8*)(dst + ks1[i]) = codes8<E4M3>(kc[i].z, kc[i].w);
    }
    if (wave == 0 && lane < 4) {
      lds.ks[u & 3][lane] = no_page ? __builtin_nanf("") : scale_k;
      lds.lvs[u & 3][lane] = log2_(scale_v);
      lds.ivs[u & 3][lane] = scale_v == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(scale_v);  // unwritten
    }
  };
  auto stage_v = [&](int u) {
    uint16_t* dst = &lds.v[u & 1][0][0];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      if (E4M3) {
        // A page before every row's window may be any, and its e4m3 codes NaN, which a weight of 0
        // would not take out; so may page 0, read for an entry outside the pool, for rows before it.
        const int t = tile_at(u) + vt[i];
        if (no_v[i] || (a.window > 0 && t + g.page - 1 <= pfirst - a.window && t >= a.sinks))
          vc[i] = u4{0, 0, 0, 0};
      }
      *(h8*)(dst + vs0[i]) = codes8<E4M3>(vc[i].x, vc[i].y);
      *(h8*)(dst + vs1[i]) = codes8<E4M3>(vc[i].z, vc[i].w);
    }
  };
  // The tail, straight to the LDS: rows behind the last token are 0, never what lies there.
  auto stage_tail = [&] {
    const int64_t base = ((int64_t)b * g.nkv + h) * g.page * HD;
    const int have = n - sp.nq;
    for (int c = tid; c < kTile * (HD / 8); c += kThreads) {
      const int r = c / (HD / 8), cc = c % (HD / 8);
      h8 k = {}, v = {};
      if (r < have) {
        k = *(const h8*)(a.pool.k_tail + base + r * HD + cc * 8);
        v = *(const h8*)(a.pool.v_tail + base + r * HD + cc * 8);
      }
      *(h8*)&lds.k[0][r][k_chunk<HD>(r, cc) * 8] = k;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = cc * 8 + i;
        lds.v[0][d][v_chunk(d, r / 8) * 8 + (r & 7)] = h_bits(v[i]);
      }
    }
    if (tid < 4) {
      lds.ks[0][tid] = 1.0f;
      lds.lvs[0][tid] = 0.0f;
      lds.ivs[0][tid] = 1.0f;
    }
  };

  // K row of this lane in a tile of 32: the scores of a lane are then tokens 8 hh ... + 7 of
  // either half
  const int krow = (n32 & 16) | (n32 & 4) << 1 | (n32 & 8) >> 1 | (n32 & 3);
  // LDS offsets (values) of this lane's chunks: a K row's k-steps, a V row's
  int ko[KS], vo[4];
#pragma unroll
  for (int i = 0; i < KS; ++i) ko[i] = krow * HD + k_chunk<HD>(krow, 2 * i + hh) * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) vo[k] = n32 * kTile + v_chunk(n32, 2 * k + hh) * 8;

  f16v s[2];
  h8 p[4];
  auto scores = [&](int u) {
    const uint16_t* kb = &lds.k[u & 1][0][0];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const h8 k = *(const h8*)(kb + t * 32 * HD + ko[i]);
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[i], i ? s[t] : f16v{}, 0, 0, 0);
      }
  };
  // What a tile is to the wavefront's rows: nothing (behind them all, or before their windows),
  // seen by all of them, or in part.
  auto nothing = [&](int t0) {
    return t0 > wlast ||
           (a.window > 0 && t0 + kTile - 1 <= wfirst - a.window && t0 >= a.sinks);
  };
  auto whole = [&](int t0, int end) {
    return t0 + kTile <= end && t0 + kTile - 1 <= wfirst &&
           (a.window <= 0 || t0 > wlast - a.window || t0 + kTile <= a.sinks);
  };
  auto soften = [&](int u, int t0, int end) {
    const bool masked = !whole(t0, end);
    // A group of 16 tokens has one scale: its largest t is that of its largest score.
    float ga[4], gb[4], gi[4], top = kNegInf;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ga[k] = lds.ks[u & 3][k] * qs;
      gb[k] = lds.lvs[u & 3][k];
      gi[k] = lds.ivs[u & 3][k];
    }
    if (masked) {
      // bit j: token t0 + j is there and seen
      uint64_t see = low_bits((end < pos + 1 ? end : pos + 1) - t0);
      if (a.window > 0)
        see &= ~low_bits(pos + 1 - a.window - t0) | low_bits(a.sinks - t0);
      see >>= hh * 8;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t bits = (uint32_t)(see >> (16 * k)) & 255u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s[k / 2][(k & 1) * 8 + i] = bits >> i & 1 ? s[k / 2][(k & 1) * 8 + i] : kNegInf;
        // scales that nothing sees may be anything; and -inf times one stays -inf
        ga[k] = bits == 0 ? 1.0f : ga[k] < 0x1p-100f ? 0x1p-100f : ga[k];
        gb[k] = bits == 0 ? 0.0f : gb[k];
        gi[k] = bits == 0 ? 0.0f : gi[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        x = fmaxf(fmaxf(x, s[k / 2][(k & 1) * 8 + i]), s[k / 2][(k & 1) * 8 + i + 1]);
      top = fmaxf(top, __builtin_fmaf(x, ga[k], gb[k]));
    }
    top = fmaxf(top, other_half(top));
    if (__ballot(top > mx + (kLift + kSlack))) {
      const float to = top > mx + (kLift + kSlack) ? top - kLift : mx;
      const float f = to > mx ? exp2_(mx - to) : 1.0f;
      mx = to;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    const float base = mx == kNegInf ? 0.0f : mx;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float sum = 0.0f;
      const float off = gb[k] - base;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = exp2_(__builtin_fmaf(s[k / 2][(k & 1) * 8 + i], ga[k], off));
        sum += w;
        p[k][i] = (_Float16)w;
      }
      l = __builtin_fmaf(sum, gi[k], l);
    }
  };
  auto values = [&](int u) {
    const uint16_t* vb = &lds.v[u & 1][0][0];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const h8 v = *(const h8*)(vb + d * 32 * kTile + vo[k]);
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[k], acc[d], 0, 0, 0);
      }
  };

  if (quant > 0) {
    // K of tiles 0 and 1 and V of tile 0 to the LDS, K of 2 and V of 1 on their way
    pages_k(0);
    pages_v(0);
    fetch_k();
    fetch_v();
    pages_k(1);
    pages_v(1);
    stage_k(0);
    stage_v(0);
    fetch_k();
    fetch_v();
    pages_k(2);
    pages_v(2);
    stage_k(1);
    fetch_k();
    pages_k(3);
    turn();
    if (!nothing(tile_at(0))) scores(0);
    turn();
    for (int u = 0; u < quant; ++u) {
      // K of u + 2 takes the place of u's, whose scores are done; V of u + 1 that of u - 1
      stage_k(u + 2);
      stage_v(u + 1);
      fetch_k();
      fetch_v();
      pages_k(u + 4);
      pages_v(u + 3);
      const int t0 = tile_at(u);
      if (!nothing(t0)) {
        soften(u, t0, sp.nq);
        values(u);
      }
      if (u + 1 < quant && !nothing(tile_at(u + 1))) scores(u + 1);
      turn();
    }
  }
  if (plast >= sp.nq && n > sp.nq && slice == slices - 1) {
    stage_tail();
    turn();
    if (wlast >= sp.nq) {
      scores(0);
      soften(0, sp.nq, n);
      values(0);
    }
  }

  l += other_half(l);
  if (!ok) return;
  const int64_t at = (int64_t)(q0 + tok) * g.nh + head;
  if (slices > 1) {  // q8_merge_kernel joins the slices
    const int64_t part = (int64_t)slice * a.total_q * g.nh + at;
    if (hh == 0) {
      a.part_ml[2 * part] = mx;
      a.part_ml[2 * part + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f4*)(a.part_acc + part * HD + d * 32 + i * 8 + hh * 4) =
            f4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (a.lse && hh == 0) a.lse[at] = l == 0.0f ? kNegInf : (mx + log2_(l)) / kLog2e;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store4(a, at * HD + d * 32 + i * 8 + hh * 4,
             f4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]} * inv);
}

// Joins the slices of every row, in their order: a thread per 4 channels.
template <int HD>
__global__ __launch_bounds__(256) void q8_merge_kernel(Geo g, AttendArgs a) {
  static_assert(256 / (HD / 4) == 1 << merge_log2(HD), "rows of a workgroup");
  const Place p = place_of(g, a, blockIdx.x, g.nh, merge_log2(HD));
  const int slices = prefill_slices(a, p.n);
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
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  store4(a, at * HD + ch, acc * inv);
  if (a.lse && ch == 0) a.lse[at] = l == 0.0f ? kNegInf : (mx + log2_(l)) / kLog2e;
}

template <int HD, bool E4M3>
static hipError_t prefill_codes(const Geo& g, const AttendArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.tiles * g.nkv), a.slices);
  if (sizeof(Lds<HD>) > 65536) {  // past 64 KiB a kernel asks for its LDS
    const hipError_t e = hipFuncSetAttribute((const void*)q8_prefill_kernel<HD, E4M3>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)sizeof(Lds<HD>));
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((q8_prefill_kernel<HD, E4M3>), grid, dim3(kThreads), sizeof(Lds<HD>), s, g, a);
  if (a.slices > 1) hipLaunchKernelGGL((q8_merge_kernel<HD>), dim3(a.merges), dim3(256), 0, s, g, a);
  return hipGetLastError();
}

hipError_t launch_prefill(const Geo& g, const AttendArgs& a, hipStream_t s) {
  const bool e = g.codes == JACQ_Q8_E4M3;
  if (g.hd == 128) return e ? prefill_codes<128, true>(g, a, s) : prefill_codes<128, false>(g, a, s);
  return e ? prefill_codes<64, true>(g, a, s) : prefill_codes<64, false>(g, a, s);
}

}  // namespace q8
}  // namespace jacq
