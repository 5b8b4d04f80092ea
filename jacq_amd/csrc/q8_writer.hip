// q8_writer.hip -- append to the 8-bit paged cache, and reading it back.
//
// Append: a workgroup per (sequence, kv head, block that the new tokens touch);
// none waits for another.  The workgroup of the first block also owns the tail:
// it has read the rows that the block takes in before it writes the rows that
// remain.  One half of its wavefronts has K, the other V, all rows in registers
// (lane = NI consecutive tokens x 8 channels), so the largest magnitude is one
// pass, a row of K codes leaves as it came, and the lane already holds NI
// consecutive tokens of each channel for the transposed V.
//
// Bound by latency: a prompt of 8191 tokens (8 kv heads of 128, e4m3, 50 MB)
// takes 13 us, 3.9 TB/s; a token for each of 64 sequences 4 us, three dependent
// rounds of memory.  Reading the same prompt back takes 12 us, 64 sequences'
// last 16 tokens 6.
#include "q8_common.h"

namespace jacq {
namespace q8 {

// 8 new or held values as fp16; what is past fp16 is infinite here, and saturated by `finite`.
__device__ inline u4 as_half(u4 raw, bool bf16) {
  if (!bf16) return raw;
  u4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h2 x = {(_Float16)__uint_as_float(raw[i] << 16),
                  (_Float16)__uint_as_float(raw[i] & 0xffff0000u)};
    r[i] = __builtin_bit_cast(uint32_t, x);
  }
  return r;
}

typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// The largest magnitude of fp16 pairs, as bits: past 0x7c00 there is a NaN, at 0x7c00 an infinity.
__device__ inline uint32_t magnitude2(uint32_t m, uint32_t x) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(us2, m),
                                                      __builtin_bit_cast(us2, x & 0x7fff7fffu)));
}
__device__ inline uint32_t magnitude8(u4 x) {
  const uint32_t m = magnitude2(magnitude2(magnitude2(magnitude2(0, x.x), x.y), x.z), x.w);
  const uint32_t lo = m & 0xffffu, hi = m >> 16;
  return lo > hi ? lo : hi;
}

// Infinities become fp16's largest.
__device__ inline u4 finite(u4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = x[i];
    if ((w & 0x7fffu) == 0x7c00u) w -= 1;
    if ((w & 0x7fff0000u) == 0x7c000000u) w -= 0x10000u;
    x[i] = w;
  }
  return x;
}

// Every lane of a row of CH lanes side by side: has one of them its bit in `lanes`?
template <int CH>
__device__ inline bool row_in(uint64_t lanes, int lane) {
  return (lanes >> (lane / CH * CH) & (((uint64_t)1 << CH) - 1)) != 0;
}

// The quotient top x / a, rounded so that every tie between codes is seen as one: n = top x is
// exact, and one residual step corrects n * (1 / a) to the quotient itself wherever that has few
// bits (a half code does).
__device__ inline float quotient(float n, float a, float inv) {
  const float q = n * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, a, n), inv, q);
}

template <bool E4M3>
__device__ inline uint32_t code4(float y0, float y1, float y2, float y3) {
  if constexpr (E4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, w, true);
  } else {
    // 2^23 + 128 + y: the sum rounds half to even to a whole number, whose low byte is the code
    const float m = 8388736.0f;
    const uint32_t a = __float_as_uint(y0 + m), b = __float_as_uint(y1 + m);
    const uint32_t c = __float_as_uint(y2 + m), d = __float_as_uint(y3 + m);
    const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);  // bytes 0c: zero
    const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return ab | cd;
  }
}

__device__ inline float half_at(u4 x, int i) {
  const uint32_t w = x[i / 2];  // by value, as in h_bits
  const h2 p = __builtin_bit_cast(h2, w);
  return (float)(i & 1 ? p.y : p.x);
}

// Codes of K: a lane's 8 channels of a token are 8 bytes of its row.
template <int HD, int NI, bool E4M3>
__device__ inline void store_k(uint8_t* dst, const u4 (&x)[NI], float a, bool poisoned) {
  constexpr float top = E4M3 ? 448.0f : 127.0f;
  const float inv = 1.0f / a;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float y[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) y[c] = quotient(half_at(x[i], c) * top, a, inv);
    u2 w = {code4<E4M3>(y[0], y[1], y[2], y[3]), code4<E4M3>(y[4], y[5], y[6], y[7])};
    if (poisoned) w = E4M3 ? u2{0, 0} : u2{0x80808080u, 0x80808080u};  // zeros: the scale is NaN
    *(u2*)(dst + i * HD) = w;
  }
}

// Codes of V: a lane's NI tokens of a channel are NI bytes of that channel's row.
template <int P, int NI, bool E4M3>
__device__ inline void store_v(uint8_t* dst, const u4 (&x)[NI], float a) {
  constexpr float top = E4M3 ? 448.0f : 127.0f;
  const float inv = 1.0f / a;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    float y[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NI; ++i) y[i] = quotient(half_at(x[i], c) * top, a, inv);
    const uint32_t w = code4<E4M3>(y[0], y[1], y[2], y[3]);
    if constexpr (NI == 2) *(uint16_t*)(dst + c * P) = (uint16_t)w;
    else *(uint32_t*)(dst + c * P) = w;
  }
}

// How a block is dealt: NI tokens a lane, PARTS wavefronts for K and as many for V.
template <int HD, int P>
struct Deal {
  static constexpr int CH = HD / 8;  // lanes of a token row
  static constexpr int NI = P * HD / 512 < 4 ? P * HD / 512 : 4;
  static constexpr int PARTS = P * HD / 512 / NI;
  static constexpr int THREADS = 128 * PARTS;
};

// blockIdx.x: kv head + NKV * block from the sequence's first touched one; blockIdx.y: sequence.
template <int HD, int P, bool E4M3>
__global__ __launch_bounds__((Deal<HD, P>::THREADS)) void q8_append_kernel(Geo g, AppendArgs a) {
  typedef Deal<HD, P> D;
  constexpr int CH = D::CH, NI = D::NI, PARTS = D::PARTS;
  constexpr float top = E4M3 ? 448.0f : 127.0f;
  __shared__ uint32_t most[2 * PARTS];             // largest magnitudes, as bits
  __shared__ uint64_t bad[2][PARTS][NI];           // lanes with a NaN
  __shared__ uint32_t mended[2 * PARTS];
  const int b = blockIdx.y, h = blockIdx.x % g.nkv, j = blockIdx.x / g.nkv;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const bool is_v = wave >= PARTS;
  const int part = is_v ? wave - PARTS : wave;
  int row0 = b, n = 1;
  if (a.cu) {
    int lo = a.cu[b], hi = a.cu[b + 1];
    lo = lo < 0 ? 0 : lo > a.total ? a.total : lo;
    hi = hi < lo ? lo : hi > a.total ? a.total : hi;
    row0 = lo;
    n = hi - lo > a.max_new ? a.max_new : hi - lo;
  }
  const int start = uniform(a.start[b]);
  const int cap = g.max_pages * P;
  if (start < 0 || start >= cap) return;
  n = uniform(n > cap - start ? cap - start : n);
  if (n < 1) return;
  const int off = start % P, first = start / P;
  const int done = (off + n) / P;  // blocks that become full
  if (j > 0 && j >= done) return;
  const int ch = lane % CH * 8;
  const uint16_t* nk = a.new_k + (int64_t)row0 * a.k_stride + (int64_t)h * HD + ch;
  const uint16_t* nv = a.new_v + (int64_t)row0 * a.v_stride + (int64_t)h * HD + ch;
  const int64_t tail = ((int64_t)b * g.nkv + h) * (P * HD) + ch;
  const bool bf16 = a.bf16 != 0;

  if (done > j) {  // block first + j: the tail's rows (of the first block), then new ones
    const int t0 = part * (P / PARTS) + lane / CH * NI;
    const uint16_t* src = is_v ? nv : nk;
    const uint16_t* held_rows = is_v ? a.pool.v_tail : a.pool.k_tail;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const int page = uniform(a.tables[(int64_t)b * g.max_pages + first + j]);
    u4 x[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int t = j * P + t0 + i - off;  // new token, or a row of the tail where negative
      x[i] = *(const u4*)(t < 0 ? held_rows + tail + (t + off) * HD : src + (int64_t)t * stride);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      x[i] = as_half(x[i], bf16 && j * P + t0 + i >= off);
      const uint32_t mi = magnitude8(x[i]);
      m = mi > m ? mi : m;
      const uint64_t nans = __ballot(mi > 0x7c00u);
      if (lane == 0) bad[is_v][part][i] = nans;
    }
    m = (uint32_t)lane63(wave_prefix((int)m, Max()));
    if (lane == 0) most[wave] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int i = 0; i < 2 * PARTS; ++i) m = most[i] > m ? most[i] : m;
    const bool rare = uniform(m) >= 0x7c00;
    bool poisoned = false;
    if (__builtin_expect(rare, 0)) {
      // Infinities saturate.  A NaN in a token's K or V: its V is 0, and K's scale NaN.
      m = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (row_in<CH>(bad[0][part][i] | bad[1][part][i], lane)) x[i] = u4{0, 0, 0, 0};
        x[i] = finite(x[i]);
        const uint32_t mi = magnitude8(x[i]);
        m = mi > m ? mi : m;
      }
      for (int q = 0; q < PARTS; ++q)
        for (int i = 0; i < NI; ++i) poisoned |= (bad[0][q][i] | bad[1][q][i]) != 0;
      m = (uint32_t)lane63(wave_prefix((int)m, Max()));
      if (lane == 0) mended[wave] = m;
      __syncthreads();
    }
    uint32_t own = 0;  // this tensor's largest
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const uint32_t v = rare ? mended[is_v * PARTS + i] : most[is_v * PARTS + i];
      own = v > own ? v : own;
    }
    const float most_own = h2f_((uint16_t)own);
    const float big = most_own > kFloor ? most_own : kFloor;
    if (page >= 0 && page < g.num_pages) {
      const int64_t slot = (int64_t)page * g.nkv + h;
      if (is_v) {
        store_v<P, NI, E4M3>(a.pool.v_code + slot * (P * HD) + ch * P + t0, x, big);
        if (part == 0 && lane == 0) a.pool.v_scale[slot] = big / top;
      } else {
        store_k<HD, NI, E4M3>(a.pool.k_code + slot * (P * HD) + t0 * HD + ch, x, big, poisoned);
        if (part == 0 && lane == 0)
          a.pool.k_scale[slot] = poisoned ? __builtin_nanf("") : big / top;
      }
    }
  }
  if (j > 0) return;
  // The block in progress: all of the new tokens, or those behind the last full block.  The tail's
  // rows that a block took in have been read by all of the workgroup.
  const int left = done ? (off + n) % P : n, from = n - left, to = done ? 0 : off;
  for (int r = threadIdx.x / CH; r < left; r += D::THREADS / CH) {
    u4 k = as_half(*(const u4*)(nk + (int64_t)(from + r) * a.k_stride), bf16);
    u4 v = as_half(*(const u4*)(nv + (int64_t)(from + r) * a.v_stride), bf16);
    const uint32_t mk = magnitude8(k), mv = magnitude8(v);
    if (__ballot(mk >= 0x7c00u || mv >= 0x7c00u)) {
      const uint64_t nans = __ballot(mk > 0x7c00u || mv > 0x7c00u);
      k = finite(k);
      v = finite(v);
      if (row_in<CH>(nans, lane)) {
        k = u4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
        v = u4{0, 0, 0, 0};
      }
    }
    *(u4*)(a.pool.k_tail + tail + (to + r) * HD) = k;
    *(u4*)(a.pool.v_tail + tail + (to + r) * HD) = v;
  }
}

template <int HD, int P>
static void append_codes(const Geo& g, const AppendArgs& a, int batch, hipStream_t s) {
  // a sequence touches at most this many blocks that fill (the first counts in any case)
  const int blocks = a.max_new / P + 1;
  const dim3 grid((unsigned)g.nkv * blocks, batch);
  if (g.codes == JACQ_Q8_E4M3)
    hipLaunchKernelGGL((q8_append_kernel<HD, P, true>), grid, dim3(Deal<HD, P>::THREADS), 0, s, g, a);
  else
    hipLaunchKernelGGL((q8_append_kernel<HD, P, false>), grid, dim3(Deal<HD, P>::THREADS), 0, s, g,
                       a);
}

hipError_t launch_append(const Geo& g, const AppendArgs& a, int batch, hipStream_t s) {
  if (g.hd == 128) {
    if (g.page == 16) append_codes<128, 16>(g, a, batch, s);
    else if (g.page == 32) append_codes<128, 32>(g, a, batch, s);
    else append_codes<128, 64>(g, a, batch, s);
  } else {
    if (g.page == 16) append_codes<64, 16>(g, a, batch, s);
    else if (g.page == 32) append_codes<64, 32>(g, a, batch, s);
    else append_codes<64, 64>(g, a, batch, s);
  }
  return hipGetLastError();
}

// ---- read back ----

struct ReadArgs {
  Pool pool;
  const int32_t* starts;
  const int32_t* ends;
  const int32_t* tables;
  void* k;
  void* v;
  int batch, total, type;
};

// Rounded to the output's type once; 8 values.
__device__ inline void store8(void* p, int64_t at, const float (&x)[8], int type) {
  if (type == JACQ_Q8_FP32) {
    f4 lo = {x[0], x[1], x[2], x[3]}, hi = {x[4], x[5], x[6], x[7]};
    *(f4*)((float*)p + at) = lo;
    *(f4*)((float*)p + at + 4) = hi;
    return;
  }
  u4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = type == JACQ_Q8_BF16 ? f2bf(x[2 * i]) : f2h_(x[2 * i]);
    const uint32_t hi = type == JACQ_Q8_BF16 ? f2bf(x[2 * i + 1]) : f2h_(x[2 * i + 1]);
    w[i] = lo | hi << 16;
  }
  *(u4*)((uint16_t*)p + at) = w;
}

// One wavefront per (16 tokens of a sequence, kv head): blockIdx.x counts them, kv heads fastest.
template <int HD, bool E4M3>
__global__ __launch_bounds__(64) void q8_read_kernel(Geo g, ReadArgs a) {
  constexpr int CH = HD / 8;
  __shared__ __align__(16) uint16_t lds[16 * (HD + 8)];
  const int h = blockIdx.x % g.nkv, lane = threadIdx.x;
  const int want = blockIdx.x / g.nkv;
  // The sequence of the wanted 16, which of its 16s it is, and the rows of the sequences before.
  // A call's tokens may outnumber 32 bits: those past `total` are dropped.
  int64_t before = 0;
  int b = -1, start = 0, end = 0, group = 0;
  int groups = 0;
  for (int base = 0; base < a.batch && b < 0; base += 64) {
    int s = 0, e = 0;
    if (base + lane < a.batch) {
      e = clamp_len(g, a.ends[base + lane]);
      s = a.starts[base + lane];
      s = s < 0 ? 0 : s > e ? e : s;
    }
    const int n = e > s ? (e + 15) / 16 - s / 16 : 0;
    const int inc = wave_prefix(n, Sum()), rows = wave_prefix(e - s, Sum());
    if (const uint64_t past = __ballot(groups + inc > want && n > 0)) {
      const int l = __builtin_ctzll(past);
      b = base + l;
      start = __builtin_amdgcn_readlane(s, l);
      end = __builtin_amdgcn_readlane(e, l);
      group = want - groups - __builtin_amdgcn_readlane(inc - n, l);
      before += __builtin_amdgcn_readlane(rows - (e - s), l);
    } else {
      groups += lane63(inc);
      before += lane63(rows);
    }
  }
  if (b < 0 || before >= a.total) return;
  const int nq = end >> g.page_log2 << g.page_log2;
  {
    const int t0 = start / 16 * 16 + group * 16;
    const bool held = t0 >= nq;  // a group of 16 is in one page or in the tail
    const int in = t0 & (g.page - 1);
    float ks = 1.0f, vs = 1.0f;
    int64_t slot = 0;
    if (!held) {
      const int page = uniform(a.tables[(int64_t)b * g.max_pages + (t0 >> g.page_log2)]);
      const bool ok = page >= 0 && page < g.num_pages;
      slot = (int64_t)(ok ? page : 0) * g.nkv + h;
      ks = ok ? a.pool.k_scale[slot] : __builtin_nanf("");
      vs = ok ? a.pool.v_scale[slot] : __builtin_nanf("");
      // V: lane = a channel's 16 tokens, transposed through the LDS
      for (int d = lane; d < HD; d += 64) {
        const u4 w = *(const u4*)(a.pool.v_code + (slot * HD + d) * g.page + in);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h2 lo, hi;
          codes4<E4M3>(w[i], lo, hi);
          lds[(4 * i + 0) * (HD + 8) + d] = h_bits(lo.x);
          lds[(4 * i + 1) * (HD + 8) + d] = h_bits(lo.y);
          lds[(4 * i + 2) * (HD + 8) + d] = h_bits(hi.x);
          lds[(4 * i + 3) * (HD + 8) + d] = h_bits(hi.y);
        }
      }
    }
    __syncthreads();
    for (int r = lane / CH; r < 16; r += 64 / CH) {
      const int t = t0 + r, ch = lane % CH * 8;
      const int64_t row = before + t - start;
      if (t < start || t >= end || row >= a.total) continue;
      h8 kc, vc;
      if (held) {
        const int64_t at = (((int64_t)b * g.nkv + h) * g.page + (t - nq)) * HD + ch;
        kc = *(const h8*)(a.pool.k_tail + at);
        vc = *(const h8*)(a.pool.v_tail + at);
      } else {
        const u2 w = *(const u2*)(a.pool.k_code + (slot * g.page + in + r) * HD + ch);
        kc = codes8<E4M3>(w.x, w.y);
        vc = *(const h8*)(lds + r * (HD + 8) + ch);
      }
      float k[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        k[i] = (float)kc[i] * ks;
        v[i] = (float)vc[i] * vs;
      }
      const int64_t at = (row * g.nkv + h) * HD + ch;
      store8(a.k, at, k, a.type);
      store8(a.v, at, v, a.type);
    }
  }
}

hipError_t launch_read(const Geo& g, const Pool& p, const int32_t* starts, const int32_t* ends,
                       const int32_t* tables, int batch, int total, void* k, void* v, int type,
                       hipStream_t s) {
  const ReadArgs a = {p, starts, ends, tables, k, v, batch, total, type};
  // a sequence's tokens touch at most one group of 16 more than a 16th of them, begun ones counted
  const dim3 grid((unsigned)g.nkv * (total / 16 + 2 * batch));
#define JACQ_READ(HD, E)                                                                 \
  hipLaunchKernelGGL((q8_read_kernel<HD, E>), grid, dim3(64), 0, s, g, a)
  if (g.hd == 128) {
    if (g.codes == JACQ_Q8_E4M3) JACQ_READ(128, true);
    else JACQ_READ(128, false);
  } else {
    if (g.codes == JACQ_Q8_E4M3) JACQ_READ(64, true);
    else JACQ_READ(64, false);
  }
#undef JACQ_READ
  return hipGetLastError();
}

}  // namespace q8
}  // namespace jacq
