// q8_prefill.hip -- attention of prompts over the 8-bit cache.
//
// A workgroup has 32 kWaves query rows of one kv head (row = query token x
// head of the group), 32 a wavefront, and goes through the tiles of 64 tokens
// that any of its rows sees.  A tile's codes are converted to fp16 once and
// shared through the LDS, two tiles deep: the next one's codes are in flight
// while this one is computed.  S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16_f16; a lane's column is a query row, so its maximum, sum
// and rescaling are the lane's own (and its partner's, 32 lanes on), and the
// order in which K's rows enter makes P the next operand as it stands.
// The scales of 16 tokens are the wavefront's: t = s (ks q) + log2(vs), as in
// q8_decode.hip, where the reason is.
#include "q8_common.h"

namespace jacq {
namespace q8 {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;
constexpr float kSlack = 8.0f;  // the running maximum moves only by more than this (base 2)
constexpr float kNegInf = -__builtin_inff();

template <int HD>
struct Lds {
  uint16_t k[2][kTile][HD];    // 16-byte chunks of a row are XOR-ed with the row
  uint16_t v[2][HD][kTile];
  float ks[2][4], lvs[2][4], ivs[2][4];  // per 16 tokens: K scale, log2 and inverse of V's
};

// Where chunk c (8 values) of a row lies, so that 16 rows' same chunk covers all banks.
template <int HD>
__device__ inline int k_chunk(int row, int c) {
  return HD == 128 ? c ^ (row & 15) : c ^ (row >> 1 & 7);
}
__device__ inline int v_chunk(int d, int c) { return c ^ (d >> 1 & 7); }

template <int HD, bool E4M3>
__global__ __launch_bounds__(kThreads, 2) void q8_prefill_kernel(Geo g, AttendArgs a, int tiles) {
  constexpr int KS = HD / 16;                        // k-steps of S^T
  constexpr int DT = HD / 32;                        // channel tiles
  constexpr int KC = kTile * HD / 16 / kThreads;     // 16-code chunks of K a thread stages
  extern __shared__ __align__(16) uint8_t shared_bytes[];
  Lds<HD>& lds = *(Lds<HD>*)shared_bytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int b = blockIdx.y, h = blockIdx.x % g.nkv;
  const int rt = tiles - 1 - (int)blockIdx.x / g.nkv;  // the longest first
  int q0, m;
  queries_of(a, b, &q0, &m);
  q0 = uniform(q0);
  m = uniform(m);
  const int rows = m * g.gqa;
  if (rt * kRows >= rows) return;
  const int n = uniform(clamp_len(g, a.lens[b]));
  const int row = rt * kRows + wave * 32 + n32;
  const bool ok = row < rows;
  const int tok = ok ? row / g.gqa : 0, head = h * g.gqa + row % g.gqa;
  const int pos = ok ? n - m + tok : -1;
  // positions of the workgroup's and the wavefront's rows
  const int end_row = rows < (rt + 1) * kRows ? rows : (rt + 1) * kRows;
  const int pfirst = n - m + rt * kRows / g.gqa, plast = n - m + (end_row - 1) / g.gqa;
  const int wr0 = rt * kRows + wave * 32;
  const int wr1 = wr0 + 32 < rows ? wr0 + 32 : rows;
  const int wfirst = n - m + wr0 / g.gqa, wlast = wr0 < rows ? n - m + (wr1 - 1) / g.gqa : -1;

  h8 q[KS];
  float qs = a.scale;
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
      big = fmaxf(big, __shfl_xor(big, 32));
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

  // Units: the sinks' tiles, the window's up to the last row's position, the tail.
  const Span sp(g, n, pfirst, a.window, a.sinks);
  int top = plast < 0 ? 0 : plast / kTile + 1;
  top = top > sp.tiles ? sp.tiles : top;
  const int quant = plast < 0 ? 0 : sp.ns + (top > sp.w0 ? top - sp.w0 : 0);
  const int units = quant + (plast >= sp.nq && n > sp.nq ? 1 : 0);

  // ---- staging: this thread's chunks of a tile ----
  u4 kc[KC], vc[KC];
  float scale_k = 0, scale_v = 0;
  const int per = g.page >> 4;                  // 16-token chunks of a V row in its page
  const int per_log2 = g.page_log2 - 4;
  auto page_at = [&](int t) {  // of the 16 tokens at t; -1: none
    const int last = sp.nq - 16;
    t = t < last ? t : last;
    const int p = a.tables[(int64_t)b * g.max_pages + (t >> g.page_log2)];
    return p >= 0 && p < g.num_pages ? p : -1;
  };
  // V chunk i of this thread: 16 tokens group vg of channel vd, side by side in memory
  auto v_place = [&](int i, int& vd, int& vg) {
    const int c = tid + kThreads * i;
    const int in = c & (HD * per - 1);
    vd = in >> per_log2;
    vg = (c / HD >> per_log2 << per_log2) + (in & (per - 1));
  };
  int pk[KC], pv[KC], ps;
  auto fetch_pages = [&](int u) {
    const int t0 = sp.tile_of(u) * kTile;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      pk[i] = page_at(t0 + (tid + kThreads * i) / (HD / 16) / 16 * 16);
      int vd, vg;
      v_place(i, vd, vg);
      pv[i] = page_at(t0 + vg * 16);
    }
    ps = page_at(t0 + (tid & 3) * 16);
  };
  auto fetch = [&](int u) {
    const int t0 = sp.tile_of(u) * kTile;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int c = tid + kThreads * i;
      const int r = c / (HD / 16), cc = c % (HD / 16);
      const int64_t s = (int64_t)(pk[i] < 0 ? 0 : pk[i]) * g.nkv + h;
      kc[i] = *(const u4*)(a.pool.k_code + (s * g.page + ((t0 + r) & (g.page - 1))) * HD + cc * 16);
      int vd, vg;
      v_place(i, vd, vg);
      const int64_t sv = (int64_t)(pv[i] < 0 ? 0 : pv[i]) * g.nkv + h;
      vc[i] = *(const u4*)(a.pool.v_code + (sv * HD + vd) * g.page +
                           ((t0 + vg * 16) & (g.page - 1)));
    }
    const int64_t s = (int64_t)(ps < 0 ? 0 : ps) * g.nkv + h;
    scale_k = ps < 0 ? __builtin_nanf("") : a.pool.k_scale[s];
    scale_v = a.pool.v_scale[s];
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int c = tid + kThreads * i;
      const int r = c / (HD / 16), cc = c % (HD / 16);
      *(h8*)&lds.k[buf][r][k_chunk<HD>(r, 2 * cc) * 8] = codes8<E4M3>(kc[i].x, kc[i].y);
      *(h8*)&lds.k[buf][r][k_chunk<HD>(r, 2 * cc + 1) * 8] = codes8<E4M3>(kc[i].z, kc[i].w);
      int vd, vg;
      v_place(i, vd, vg);
      *(h8*)&lds.v[buf][vd][v_chunk(vd, 2 * vg) * 8] = codes8<E4M3>(vc[i].x, vc[i].y);
      *(h8*)&lds.v[buf][vd][v_chunk(vd, 2 * vg + 1) * 8] = codes8<E4M3>(vc[i].z, vc[i].w);
    }
    if (tid < 4) {
      lds.ks[buf][tid] = scale_k;
      lds.lvs[buf][tid] = log2_(scale_v);
      lds.ivs[buf][tid] = 1.0f / scale_v;
    }
  };
  // The tail, straight to the LDS: rows behind the last token are 0, never what lies there.
  auto stage_tail = [&](int buf) {
    const int64_t base = ((int64_t)b * g.nkv + h) * g.page * HD;
    const int have = n - sp.nq;
    for (int c = tid; c < kTile * (HD / 8); c += kThreads) {
      const int r = c / (HD / 8), cc = c % (HD / 8);
      h8 k = {}, v = {};
      if (r < have) {
        k = *(const h8*)(a.pool.k_tail + base + r * HD + cc * 8);
        v = *(const h8*)(a.pool.v_tail + base + r * HD + cc * 8);
      }
      *(h8*)&lds.k[buf][r][k_chunk<HD>(r, cc) * 8] = k;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = cc * 8 + i;
        lds.v[buf][d][v_chunk(d, r / 8) * 8 + (r & 7)] = h_bits(v[i]);
      }
    }
    if (tid < 4) {
      lds.ks[buf][tid] = 1.0f;
      lds.lvs[buf][tid] = 0.0f;
      lds.ivs[buf][tid] = 1.0f;
    }
  };

  f16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f16v{};
  float mx = kNegInf, l = 0.0f;
  // K row of this lane in a tile of 32: the scores of a lane are then tokens 8 hh ... + 7 of
  // either half
  const int krow = (n32 & 16) | (n32 & 4) << 1 | (n32 & 8) >> 1 | (n32 & 3);

  auto compute = [&](int buf, int t0, int end) {
    if (t0 > wlast) return;  // the wavefront's rows are all before the tile
    if (a.window > 0 && t0 + kTile - 1 <= wfirst - a.window && t0 >= a.sinks) return;
    const bool masked = t0 + kTile > end || t0 + kTile - 1 > wfirst ||
                        (a.window > 0 && t0 <= wlast - a.window && t0 + kTile > a.sinks);
    f16v s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f16v{};
      const int r = t * 32 + krow;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const h8 k = *(const h8*)&lds.k[buf][r][k_chunk<HD>(r, 2 * i + hh) * 8];
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[i], s[t], 0, 0, 0);
      }
    }
    float top = kNegInf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int grp = t * 2 + i / 8;
        s[t][i] = __builtin_fmaf(s[t][i], lds.ks[buf][grp] * qs, lds.lvs[buf][grp]);
        if (masked) {
          const int j = t0 + grp * 16 + hh * 8 + (i & 7);
          s[t][i] = j < end && sees(j, pos, a.window, a.sinks) ? s[t][i] : kNegInf;
        }
        top = fmaxf(top, s[t][i]);
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__ballot(top > mx + kSlack)) {
      const float to = top > mx + kSlack ? top : mx;
      const float f = to > mx ? exp2_(mx - to) : 1.0f;
      mx = to;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    const float base = mx == kNegInf ? 0.0f : mx;
    h8 p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = exp2_(s[k / 2][(k & 1) * 8 + i] - base);
        sum += w;
        p[k][i] = (_Float16)w;
      }
      l += sum == 0.0f ? 0.0f : sum * lds.ivs[buf][k];  // a scale that nothing sees may be any
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int r = d * 32 + n32;
        const h8 v = *(const h8*)&lds.v[buf][r][v_chunk(r, 2 * k + hh) * 8];
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[k], acc[d], 0, 0, 0);
      }
  };

  if (quant > 0) {
    fetch_pages(0);
    fetch(0);
    if (quant > 1) fetch_pages(1);
    stage(0);
  } else if (units > 0) {
    stage_tail(0);
  }
  __syncthreads();
  for (int u = 0; u < units; ++u) {
    const int buf = u & 1;
    if (u + 1 < quant) {
      fetch(u + 1);
      if (u + 2 < quant) fetch_pages(u + 2);
    }
    if (u < quant) compute(buf, sp.tile_of(u) * kTile, sp.nq);
    else compute(buf, sp.nq, n);
    if (u + 1 < quant) stage(buf ^ 1);
    else if (u + 1 < units) stage_tail(buf ^ 1);
    __syncthreads();
  }

  l += __shfl_xor(l, 32);
  if (!ok) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = ((int64_t)(q0 + tok) * g.nh + head) * HD;
  if (a.lse && hh == 0)
    a.lse[(int64_t)(q0 + tok) * g.nh + head] = l == 0.0f ? kNegInf : (mx + log2_(l)) / kLog2e;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ch = d * 32 + i * 8 + hh * 4;
      const f4 x = {acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv, acc[d][4 * i + 2] * inv,
                    acc[d][4 * i + 3] * inv};
      if (a.o_type == JACQ_Q8_FP32) {
        *(f4*)((float*)a.o + at + ch) = x;
      } else {
        const bool bf = a.o_type == JACQ_Q8_BF16;
        const uint32_t x0 = bf ? f2bf(x.x) : f2h_(x.x), x1 = bf ? f2bf(x.y) : f2h_(x.y);
        const uint32_t x2 = bf ? f2bf(x.z) : f2h_(x.z), x3 = bf ? f2bf(x.w) : f2h_(x.w);
        *(u2*)((uint16_t*)a.o + at + ch) = u2{x0 | x1 << 16, x2 | x3 << 16};
      }
    }
}

hipError_t launch_prefill(const Geo& g, const AttendArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.max_q * g.gqa;
  const int tiles = (int)((rows + kRows - 1) / kRows);
  const dim3 grid((unsigned)tiles * g.nkv, a.batch);
#define JACQ_PREFILL(HD, E)                                                                  \
  hipLaunchKernelGGL((q8_prefill_kernel<HD, E>), grid, dim3(kThreads), sizeof(Lds<HD>), s, g, a, \
                     tiles)
  if (g.hd == 128) {
    if (g.codes == JACQ_Q8_E4M3) JACQ_PREFILL(128, true);
    else JACQ_PREFILL(128, false);
  } else {
    if (g.codes == JACQ_Q8_E4M3) JACQ_PREFILL(64, true);
    else JACQ_PREFILL(64, false);
  }
#undef JACQ_PREFILL
  return hipGetLastError();
}

}  // namespace q8
}  // namespace jacq
