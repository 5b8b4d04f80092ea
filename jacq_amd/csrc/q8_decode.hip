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
// so the P that is rounded to fp16 is at most 2^kSlack, however the scales
// differ between blocks, and no accumulator needs a scale of its own.
// (fp16 holds w to 2^-12; bf16 would hold it to 2^-9.)
#include "q8_common.h"

namespace jacq {
namespace q8 {

constexpr int kWaves = 4;         // wavefronts of a workgroup: they share a run, unit by unit
constexpr float kSlack = 8.0f;    // the running maximum moves only by more than this (base 2)
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
      pos[nb] = ok ? s.span.n - s.m + tok : -1;
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
  __device__ int64_t slot_of(const Segment& s, int page) const {
    return (int64_t)(exists(page) ? page : 0) * g.nkv + s.h;
  }

  __device__ void pages(const Segment& s, int tile, int& pk, int& pv) const {
    pk = page_of(s, tile * kTile + n16 / 4 * 16);
    pv = page_of(s, tile * kTile + kq * 16);
  }

  // A quantised tile's K codes with the scales, and its V codes.
  __device__ void load_k(const Segment& s, int tile, int pk, int pv, Codes& c) const {
    const int tk = (tile * kTile + n16 / 4 * 16) & (g.page - 1);
    const int64_t sk = slot_of(s, pk), sv = slot_of(s, pv);
    const uint8_t* k = a.pool.k_code + (sk * g.page + tk + (n16 & 3)) * HD + kq * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < KL; ++j) c.k[t][j] = *(const u4*)(k + t * 4 * HD + j * 64);
    c.ks = a.pool.k_scale[sv];
    c.there = exists(pv);
    c.vs = a.pool.v_scale[sv];
  }
  __device__ void load_v(const Segment& s, int tile, int pv, Codes& c) const {
    const int tv = (tile * kTile + kq * 16) & (g.page - 1);
    const int64_t sv = slot_of(s, pv);
    const uint8_t* v = a.pool.v_code + (sv * HD + n16) * g.page + tv;
#pragma unroll
    for (int d = 0; d < DT; ++d) c.v[d] = *(const u4*)(v + d * 16 * g.page);
  }

  // Scores -> weights -> O^T.  sc: raw scores of this lane's 16 tokens, t0 their first one;
  // tokens from `end` on are not there.  Returns through pv_step the fp16 weights.
  __device__ void soften(const Segment& s, int nb, f4 (&sc)[4], int t0, int end, float ks, float vs,
                         bool masked, bool weigh, h8& p0, h8& p1) {
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
    if (__ballot(mx > m[nb] + kSlack)) {  // also where m is -inf and mx is not
      const float to = mx > m[nb] + kSlack ? mx : m[nb];
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
    if (weigh && t0 < end && nb * 16 + n16 < s.nrows) {
      const int64_t seg = ((int64_t)s.b * g.nkv + s.h) * a.row_blocks + s.rb;
      a.group_lse[(seg * a.groups + (t0 >> 4)) * a.rows + nb * 16 + n16] = base + log2_(part);
    }
  }

  __device__ bool needs_mask(const Segment& s, int t0, int end) const {
    // uniform: the tile's 64 tokens are all there and every row sees them
    const int first = s.span.n - s.m + s.rb * 16 * NB / g.gqa;
    const int last = s.span.n - s.m + (s.rb * 16 * NB + s.nrows - 1) / g.gqa;
    return t0 + kTile > end || t0 + kTile - 1 > first ||
           (a.window > 0 && t0 <= last - a.window && t0 + kTile > a.sinks);
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
      soften(s, nb, sc[nb], s.span.nq + kq * 16, s.span.n, 1.0f, 1.0f, true, a.weights != nullptr,
             p[nb][0], p[nb][1]);
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
      if (d & 1) __builtin_amdgcn_sched_barrier(0);  // two channel tiles' loads at a time
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
      load_k(s, tile, pk, pv, c);
      load_v(s, tile, pv, c);
      if (u0 + kWaves < e) pages(s, sp.tile_of(u0 + kWaves), nk, nv);
      for (;;) {
        const int next = u0 + kWaves < e ? sp.tile_of(u0 + kWaves) : -1;
        const int t0 = tile * kTile;
        const bool masked = needs_mask(s, t0, sp.nq);
        f4 sc[NB][4];
        scores(c, sc);
        const float ks = c.there ? c.ks : __builtin_nanf(""), vs = c.vs;
        if (next >= 0) load_k(s, next, nk, nv, c);
        h8 p[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          soften(s, nb, sc[nb], t0 + kq * 16, sp.nq, ks, vs, masked, a.weights != nullptr,
                 p[nb][0], p[nb][1]);
        values(c, p);
        u0 += kWaves;
        if (next < 0) break;
        load_v(s, next, nv, c);
        if (u0 + kWaves < e) pages(s, sp.tile_of(u0 + kWaves), nk, nv);
        tile = next;
      }
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

// The stream: all segments' units one after another, sequence by sequence, cut into `runs` equal
// runs of at least min_units.  Segment x of the stream starts at `first`.
struct Stream {
  int64_t total;
  int runs;
  __device__ int64_t begin(int r) const { return total * r / runs; }
  __device__ int run_of(int64_t unit) const {  // the run that holds it
    int r = (int)(((unit + 1) * runs - 1) / total);
    while (r + 1 < runs && begin(r + 1) <= unit) ++r;
    while (r > 0 && begin(r) > unit) --r;
    return r;
  }
};

template <int ROWS>
__device__ inline void sequence_span(const Geo& g, const AttendArgs& a, int b, int* q0, int* m,
                                     Span* span, int64_t* units) {
  queries_of(a, b, q0, m);
  const int n = clamp_len(g, a.lens[b]);
  *span = Span(g, n, n - *m, a.window, a.sinks);
  const int blocks = (*m * g.gqa + ROWS - 1) / ROWS;
  *units = (int64_t)span->units * blocks * g.nkv;
}

// Total units of the batch (over the lanes of one wavefront), and the sequence that holds `unit`
// with the units before it; unit < 0 only totals.
template <int ROWS>
__device__ inline int64_t scan(const Geo& g, const AttendArgs& a, int lane, int64_t unit, int* seq,
                               int64_t* before) {
  int64_t sum = 0;
  for (int base = 0; base < a.batch; base += 64) {
    int64_t u = 0;
    if (base + lane < a.batch) {
      int q0, m;
      Span sp;
      sequence_span<ROWS>(g, a, base + lane, &q0, &m, &sp, &u);
    }
    int64_t inc = u;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t x = __shfl_up(inc, d);
      if (lane >= d) inc += x;
    }
    const uint64_t past = __ballot(sum + inc > unit && u > 0);
    if (unit >= 0 && past) {
      const int l = __builtin_ctzll(past);
      *seq = base + l;
      *before = sum + __shfl(inc - u, l);
      return sum;  // not the total: the caller has it
    }
    sum += __shfl(inc, 63);
  }
  return sum;
}

// Workgroups of kWaves wavefronts.  runs > 0: run blockIdx.x of the stream; else the segment
// blockIdx.x = (sequence, kv head, row block) whole.
template <int HD, bool E4M3, int NB>
__global__ __launch_bounds__(64 * kWaves, NB == 1 ? 2 : 1) void q8_decode_kernel(Geo g,
                                                                                 AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  constexpr int LD = HD + 4;
  __shared__ __align__(16) float red[kWaves][ROWS][LD];
  __shared__ float ml[kWaves][ROWS][2];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Wave<HD, E4M3, NB> w(g, a, lane);

  Stream st;
  int64_t at, end;  // units left of this workgroup's run
  Segment s;
  int64_t seg0;     // the sequence's first unit
  int run = blockIdx.x;
  if (a.runs) {
    st.total = scan<ROWS>(g, a, lane, -1, nullptr, nullptr);
    int64_t most = (st.total + a.min_units - 1) / a.min_units;
    st.runs = (int)(most < a.runs ? most : a.runs);
    if (run >= st.runs) return;
    at = st.begin(run);
    end = st.begin(run + 1);
    scan<ROWS>(g, a, lane, at, &s.b, &seg0);
    s.b = uniform(s.b);
  } else {
    s.b = blockIdx.x / (g.nkv * a.row_blocks);
    seg0 = at = 0;
    end = 1;
  }

  while (at < end) {
    int64_t units;
    sequence_span<ROWS>(g, a, s.b, &s.q0, &s.m, &s.span, &units);
    const int blocks = (s.m * g.gqa + ROWS - 1) / ROWS;
    int u0, u1;
    bool whole;
    if (a.runs) {
      if (blocks == 0 || at >= seg0 + units) {  // on to the next sequence
        seg0 += units;
        ++s.b;
        continue;
      }
      const int x = (int)((at - seg0) / s.span.units);
      s.h = uniform(x / blocks);
      s.rb = uniform(x % blocks);
      const int64_t first = seg0 + (int64_t)x * s.span.units;
      u0 = uniform((int)(at - first));
      const int64_t e = end - first;
      u1 = uniform(e < s.span.units ? (int)e : s.span.units);
      whole = u0 == 0 && u1 == s.span.units;
      at = first + u1;
    } else {
      const int x = blockIdx.x % (g.nkv * a.row_blocks);
      s.h = x / a.row_blocks;
      s.rb = x % a.row_blocks;
      if (s.rb >= blocks) return;
      u0 = 0;
      u1 = s.span.units;
      whole = true;
      at = end;
    }
    const int left = s.m * g.gqa - s.rb * ROWS;
    s.nrows = left < ROWS ? left : ROWS;
    w.start(s);
    w.units(s, u0 + wave, u1);

    // Fold the wavefronts' pieces: each leaves (m, l, acc) as they are, the reader scales.
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
        // a piece without a maximum saw nothing, or only NaN: l tells
        const float mv = ml[v][row][0];
        const float f = mv == kNegInf ? 1.0f : exp2_(mv - mm);
        l += ml[v][row][1] * f;
#pragma unroll
        for (int c = 0; c < PER; ++c) x[c] += red[v][row][ch + c] * f;
      }
      if (whole) {
        finish_row(g, a, s, row, HD, ch, x, PER, l, mm);
      } else {
        const int64_t slot = (int64_t)2 * run + (u0 > 0 ? 0 : 1);
        float* dst = a.part_acc + (slot * a.rows + row) * HD + ch;
#pragma unroll
        for (int c = 0; c < PER; c += 4) *(f4*)(dst + c) = *(f4*)(x + c);
        if (ch == 0) {
          a.part_ml[(slot * a.rows + row) * 2] = mm;
          a.part_ml[(slot * a.rows + row) * 2 + 1] = l;
        }
      }
    }
    __syncthreads();  // the fold's LDS, before the next piece's
  }
}

// Joins the pieces of the segments that runs cut, in the order of the runs.  blockIdx.x: segment,
// blockIdx.y: row.
template <int HD, int NB>
__global__ __launch_bounds__(256) void q8_join_kernel(Geo g, AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  constexpr int TC = HD / 4;      // threads of a piece's row
  constexpr int PG = 256 / TC;    // pieces at a time
  __shared__ __align__(16) float red[PG][HD];
  __shared__ float ml[PG][2];
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  Segment s;
  s.b = blockIdx.x / (g.nkv * a.row_blocks);
  const int x = blockIdx.x % (g.nkv * a.row_blocks);
  int64_t units, before = 0, total = 0;
  // the units of the sequences before b, and of all
  for (int base = 0; base < a.batch; base += 64) {
    int64_t u = 0;
    if (base + lane < a.batch) {
      int q0, m;
      Span sp;
      sequence_span<ROWS>(g, a, base + lane, &q0, &m, &sp, &u);
    }
    int64_t v = base + lane < s.b ? u : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      u += __shfl_xor(u, d);
      v += __shfl_xor(v, d);
    }
    total += u;
    before += v;
  }
  sequence_span<ROWS>(g, a, s.b, &s.q0, &s.m, &s.span, &units);
  const int blocks = (s.m * g.gqa + ROWS - 1) / ROWS;
  // row blocks of the grid that this sequence lacks have nothing to do
  s.h = x / a.row_blocks;
  s.rb = x % a.row_blocks;
  if (s.rb >= blocks) return;
  const int left = s.m * g.gqa - s.rb * ROWS;
  s.nrows = left < ROWS ? left : ROWS;
  if (row >= s.nrows) return;
  Stream st;
  st.total = total;
  const int64_t most = (total + a.min_units - 1) / a.min_units;
  st.runs = (int)(most < a.runs ? most : a.runs);
  const int64_t first = before + (int64_t)(s.h * blocks + s.rb) * s.span.units;
  const int r0 = st.run_of(first), r1 = st.run_of(first + s.span.units - 1);
  if (r0 == r1) return;  // one run had all of it
  const int grp = threadIdx.x / TC, c = threadIdx.x % TC * 4;
  float mm = kNegInf, l = 0.0f;
  f4 acc = {0, 0, 0, 0};
  for (int r = r0 + grp; r <= r1; r += PG) {
    const int64_t slot = (int64_t)2 * r + (st.begin(r) > first ? 0 : 1);
    const float pm = a.part_ml[(slot * a.rows + row) * 2];
    const float pl = a.part_ml[(slot * a.rows + row) * 2 + 1];
    const f4 pa = *(const f4*)(a.part_acc + (slot * a.rows + row) * HD + c);
    const float to = fmaxf(mm, pm);
    const float f0 = mm == kNegInf ? 1.0f : exp2_(mm - to);
    const float f1 = pm == kNegInf ? 1.0f : exp2_(pm - to);
    acc = acc * f0 + pa * f1;
    l = l * f0 + pl * f1;
    mm = to;
  }
  *(f4*)&red[grp][c] = acc;
  if (c == 0) {
    ml[grp][0] = mm;
    ml[grp][1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= TC) return;
  mm = kNegInf;
  for (int i = 0; i < PG; ++i) mm = fmaxf(mm, ml[i][0]);
  l = 0.0f;
  float o[4] = {0, 0, 0, 0};
  for (int i = 0; i < PG; ++i) {
    const float f = ml[i][0] == kNegInf ? 1.0f : exp2_(ml[i][0] - mm);
    l += ml[i][1] * f;
    for (int k = 0; k < 4; ++k) o[k] += red[i][c + k] * f;
  }
  finish_row(g, a, s, row, HD, c, o, 4, l, mm);
}

// Adds up the weight of every block: a thread per 16 tokens, over kv heads, row blocks and rows in
// that order; then the 16s of a page.  blockIdx.y: sequence.
template <int NB>
__global__ __launch_bounds__(256) void q8_weights_kernel(Geo g, AttendArgs a) {
  constexpr int ROWS = 16 * NB;
  const int b = blockIdx.y, grp = blockIdx.x * 256 + threadIdx.x;
  int q0, m;
  Span sp;
  int64_t units;
  sequence_span<ROWS>(g, a, b, &q0, &m, &sp, &units);
  const int blocks = (m * g.gqa + ROWS - 1) / ROWS;
  const int t0 = grp * 16, tile = t0 / kTile;
  // groups that no unit covers were not written by this call
  const bool there = t0 < sp.n && m > 0 && (t0 >= sp.nq || tile < sp.ns || tile >= sp.w0);
  float sum = 0.0f;
  if (there) {
    for (int h = 0; h < g.nkv; ++h)
      for (int rb = 0; rb < blocks; ++rb) {
        const int64_t seg = ((int64_t)b * g.nkv + h) * a.row_blocks + rb;
        const float* src = a.group_lse + (seg * a.groups + grp) * a.rows;
        const int left = m * g.gqa - rb * ROWS, rows = left < ROWS ? left : ROWS;
        for (int r = 0; r < rows; ++r) {
          const int x = rb * ROWS + r;
          const float lse = a.row_lse[(int64_t)(q0 + x / g.gqa) * g.nh + h * g.gqa + x % g.gqa];
          if (lse != kNegInf) sum += exp2_(src[r] - lse);
        }
      }
  }
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
  const unsigned blocks = a.runs ? a.runs : segments;
  hipLaunchKernelGGL((q8_decode_kernel<HD, E4M3, NB>), dim3(blocks), dim3(64 * kWaves), 0, s, g, a);
  if (a.runs)
    hipLaunchKernelGGL((q8_join_kernel<HD, NB>), dim3(segments, a.rows), dim3(256), 0, s, g, a);
  if (a.weights)
    hipLaunchKernelGGL((q8_weights_kernel<NB>), dim3((a.groups + 255) / 256, a.batch), dim3(256), 0,
                       s, g, a);
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
