// q8_writer.hip -- append to the 8-bit paged cache, and reading it back.
//
// A wavefront per (sequence, kv head, block that the new tokens touch); none
// waits for another.  The wavefront of the first block also owns the tail: it
// reads the rows that the block takes in before it writes the rows that
// remain.  All rows of a block are in registers (lane = NI consecutive tokens
// x 8 channels), so the block's largest magnitude is one pass and a shuffle,
// a row of K codes leaves as it came, and the lane already holds NI
// consecutive tokens of each channel for the transposed V.
#include "q8_common.h"

namespace jacq {
namespace q8 {

// 8 new or held values as fp16: bf16 is converted, magnitudes saturate at fp16's largest, NaN
// stays.
__device__ inline h8 as_half(u4 raw, bool bf16) {
  h8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = raw[i / 2];
    const uint32_t b = i & 1 ? w >> 16 : w & 0xffffu;
    float f = bf16 ? bf2f(b) : h2f_((uint16_t)b);
    f = f > kHalfMax ? kHalfMax : f;
    f = f < -kHalfMax ? -kHalfMax : f;
    r[i] = (_Float16)f;
  }
  return r;
}

__device__ inline bool has_nan(h8 x) {
  bool n = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) n |= x[i] != x[i];
  return n;
}

// The token row of this lane holds a NaN in some channel of K or V: rows are CH lanes side by side.
template <int CH>
__device__ inline void couple_nan(h8& k, h8& v, int lane) {
  const uint64_t bad = __ballot(has_nan(k) || has_nan(v));
  if (__builtin_expect(bad == 0, 1)) return;
  const uint64_t row = (((uint64_t)1 << CH) - 1) << (lane / CH * CH);
  if (bad & row) {
    const _Float16 nan = __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
    k = h8{nan, nan, nan, nan, nan, nan, nan, nan};
    v = h8{};
  }
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

template <int NI>
__device__ inline float largest(const h8 (&x)[NI]) {
  float a = kFloor;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) a = fmaxf(a, __builtin_fabsf((float)x[i][c]));  // a NaN is dropped
#pragma unroll
  for (int s = 32; s; s >>= 1) a = fmaxf(a, __shfl_xor(a, s));
  return a;
}

// Codes of K: a lane's 8 channels of a token are 8 bytes of its row.
template <int HD, int P, bool E4M3>
__device__ inline void store_k(const jacq_q8_pool& pool, const h8 (&x)[P * HD / 512], int64_t slot,
                               int t0, int ch, int lane) {
  constexpr int NI = P * HD / 512;
  constexpr float top = E4M3 ? 448.0f : 127.0f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NI; ++i) nan |= x[i][0] != x[i][0];  // couple_nan fills whole rows
  const bool poisoned = __ballot(nan) != 0;
  const float a = largest(x), inv = 1.0f / a;
  uint8_t* dst = pool.k_code + slot * (P * HD) + t0 * HD + ch;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float y[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      y[c] = quotient((float)x[i][c] * top, a, inv);
      if (poisoned) y[c] = 0.0f;  // no NaN codes: the scale says it
    }
    u2 w = {code4<E4M3>(y[0], y[1], y[2], y[3]), code4<E4M3>(y[4], y[5], y[6], y[7])};
    *(u2*)(dst + i * HD) = w;
  }
  if (lane == 0) pool.k_scale[slot] = poisoned ? __builtin_nanf("") : a / top;
}

// Codes of V: a lane's NI tokens of a channel are NI bytes of that channel's row.
template <int HD, int P, bool E4M3>
__device__ inline void store_v(const jacq_q8_pool& pool, const h8 (&x)[P * HD / 512], int64_t slot,
                               int t0, int ch, int lane) {
  constexpr int NI = P * HD / 512;
  constexpr float top = E4M3 ? 448.0f : 127.0f;
  const float a = largest(x), inv = 1.0f / a;
  uint8_t* dst = pool.v_code + slot * (P * HD) + ch * P + t0;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    float y[NI < 4 ? 4 : NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) y[i] = quotient((float)x[i][c] * top, a, inv);
    if constexpr (NI == 2) {
      *(uint16_t*)(dst + c * P) = (uint16_t)code4<E4M3>(y[0], y[1], 0.0f, 0.0f);
    } else if constexpr (NI == 4) {
      *(uint32_t*)(dst + c * P) = code4<E4M3>(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int i = 0; i < NI; i += 8) {
        u2 w = {code4<E4M3>(y[i], y[i + 1], y[i + 2], y[i + 3]),
                code4<E4M3>(y[i + 4], y[i + 5], y[i + 6], y[i + 7])};
        *(u2*)(dst + c * P + i) = w;
      }
    }
  }
  if (lane == 0) pool.v_scale[slot] = a / top;
}

// blockIdx.x: kv head + NKV * block from the sequence's first touched one; blockIdx.y: sequence.
template <int HD, int P, bool E4M3>
__global__ __launch_bounds__(64) void q8_append_kernel(Geo g, AppendArgs a) {
  constexpr int CH = HD / 8;    // lanes of a token row
  constexpr int NI = P * HD / 512;  // tokens of a lane
  const int b = blockIdx.y, h = blockIdx.x % g.nkv, j = blockIdx.x / g.nkv;
  const int lane = threadIdx.x;
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
  const int t0 = lane / CH * NI, ch = lane % CH * 8;
  const uint16_t* nk = a.new_k + (int64_t)row0 * a.k_stride + (int64_t)h * HD + ch;
  const uint16_t* nv = a.new_v + (int64_t)row0 * a.v_stride + (int64_t)h * HD + ch;
  const int64_t tail = ((int64_t)b * g.nkv + h) * (P * HD) + ch;
  const bool bf16 = a.bf16 != 0;

  if (done > j) {  // block first + j: the tail's rows (of the first block), then new ones
    h8 k[NI], v[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int t = j * P + t0 + i - off;  // new token, or a row of the tail where negative
      const bool held = t < 0;
      const u4 rk = *(const u4*)(held ? a.pool.k_tail + tail + (t + off) * HD
                                      : nk + (int64_t)t * a.k_stride);
      const u4 rv = *(const u4*)(held ? a.pool.v_tail + tail + (t + off) * HD
                                      : nv + (int64_t)t * a.v_stride);
      k[i] = as_half(rk, bf16 && !held);
      v[i] = as_half(rv, bf16 && !held);
      couple_nan<CH>(k[i], v[i], lane);
    }
    const int page = uniform(a.tables[(int64_t)b * g.max_pages + first + j]);
    if (page >= 0 && page < g.num_pages) {
      const int64_t slot = (int64_t)page * g.nkv + h;
      store_k<HD, P, E4M3>(a.pool, k, slot, t0, ch, lane);
      store_v<HD, P, E4M3>(a.pool, v, slot, t0, ch, lane);
    }
  }
  if (j > 0) return;
  // The block in progress: all of the new tokens, or those behind the last full block.
  const int left = done ? (off + n) % P : n, from = n - left, to = done ? 0 : off;
  for (int r = lane / CH; r < left; r += 64 / CH) {
    h8 k = as_half(*(const u4*)(nk + (int64_t)(from + r) * a.k_stride), bf16);
    h8 v = as_half(*(const u4*)(nv + (int64_t)(from + r) * a.v_stride), bf16);
    couple_nan<CH>(k, v, lane);
    *(h8*)(a.pool.k_tail + tail + (to + r) * HD) = k;
    *(h8*)(a.pool.v_tail + tail + (to + r) * HD) = v;
  }
}

template <int HD, int P>
static void append_codes(const Geo& g, const AppendArgs& a, int batch, hipStream_t s) {
  // a sequence touches at most this many blocks that fill (the first counts in any case)
  const int blocks = a.max_new / P + 1;
  const dim3 grid((unsigned)g.nkv * blocks, batch);
  if (g.codes == JACQ_Q8_E4M3)
    hipLaunchKernelGGL((q8_append_kernel<HD, P, true>), grid, dim3(64), 0, s, g, a);
  else
    hipLaunchKernelGGL((q8_append_kernel<HD, P, false>), grid, dim3(64), 0, s, g, a);
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

// One wavefront per (kv head, 16 tokens from the sequence's first group of 16); blockIdx.y:
// sequence.  Its rows of the output start where those of the sequences before end.
template <int HD, bool E4M3>
__global__ __launch_bounds__(64) void q8_read_kernel(Geo g, ReadArgs a) {
  constexpr int CH = HD / 8;
  __shared__ __align__(16) uint16_t lds[16 * (HD + 8)];
  const int b = blockIdx.y, h = blockIdx.x % g.nkv, lane = threadIdx.x;
  int64_t before = 0;  // a call's tokens may outnumber 32 bits: what is past `total` is dropped
  int start = 0, end = 0;
  for (int base = 0; base <= b; base += 64) {
    int s = 0, e = 0;
    if (base + lane <= b) {
      e = clamp_len(g, a.ends[base + lane]);
      s = a.starts[base + lane];
      s = s < 0 ? 0 : s > e ? e : s;
    }
    int n = base + lane < b ? e - s : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
    before += n;
    if (base + 64 > b) {
      start = __shfl(s, b - base);
      end = __shfl(e, b - base);
    }
  }
  start = uniform(start);
  end = uniform(end);
  const int nq = end >> g.page_log2 << g.page_log2;
  for (int t0 = start / 16 * 16 + (int)(blockIdx.x / g.nkv) * 16; t0 < end;
       t0 += (int)(gridDim.x / g.nkv) * 16) {
    __syncthreads();
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
  // enough wavefronts for one sequence to hold all the rows; the kernel loops past them
  int groups = (total + 15) / 16 + 1;
  const int cap = 4096 / (batch < 64 ? batch : 64) + 1;
  groups = groups > cap ? cap : groups;
  const dim3 grid((unsigned)g.nkv * groups, batch);
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
