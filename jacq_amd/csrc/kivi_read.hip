// kivi_read.hip -- reading the int4 cache back.
//
// A wavefront has the 32 tokens of a group, or of the residual window, and a kv head; a lane 8 channels
// of every (64 / (HD / 8))th token.  A group's scales of K are a lane's for all its tokens.
// Bound by memory, mostly by what is written: 16 caches of 1024 to 16384 tokens, 40/8 heads of 128, to fp16
// take 154 us, as long as a copy of as many bytes (4.9 TB/s); with all the registers that the compiler likes
// to take (248, two wavefronts a SIMD) 180.
#include "kivi_attend.h"

namespace jacq {

namespace {

struct ReadArgs {
  KiviPool pool;
  const int32_t* starts;
  const int32_t* ends;
  const int32_t* tables;
  void* k;
  void* v;
  int batch, total;
};

// 8 values c * s + z, rounded to the output's type once (bf16: of the fp32 sum, which is exact
// unless the two are more than 2^9 apart).
template <int TYPE>
__device__ inline void store8(void* p, int64_t at, uint32_t w, const h2 (&s)[4], const h2 (&z)[4]) {
  const Nibbles n(w);
  const uint32_t lo = __builtin_amdgcn_perm(n.odd, n.even, 0x05010400u);
  const uint32_t hi = __builtin_amdgcn_perm(n.odd, n.even, 0x07030602u);
  const h2 c[4] = {codes_lo(lo), codes_hi(lo), codes_lo(hi), codes_hi(hi)};
  u4 out;
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (TYPE == kFp16) {
      out[i] = bits(fma2(c[i], s[i], z[i]));
    } else {
      x[2 * i] = __builtin_fmaf((float)c[i].x, (float)s[i].x, (float)z[i].x);
      x[2 * i + 1] = __builtin_fmaf((float)c[i].y, (float)s[i].y, (float)z[i].y);
      if (TYPE == kBf16) out[i] = f2bf(x[2 * i]) | (uint32_t)f2bf(x[2 * i + 1]) << 16;
    }
  }
  if (TYPE == kFp32) {
    *(f4*)((float*)p + at) = f4{x[0], x[1], x[2], x[3]};
    *(f4*)((float*)p + at + 4) = f4{x[4], x[5], x[6], x[7]};
  } else {
    *(u4*)((uint16_t*)p + at) = out;
  }
}

// 8 fp16 values as they are.
template <int TYPE>
__device__ inline void store8(void* p, int64_t at, u4 raw) {
  if (TYPE == kFp16) {
    *(u4*)((uint16_t*)p + at) = raw;
    return;
  }
  const h8 x = __builtin_bit_cast(h8, raw);
  if (TYPE == kBf16) {
    u4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      out[i] = f2bf((float)x[2 * i]) | (uint32_t)f2bf((float)x[2 * i + 1]) << 16;
    *(u4*)((uint16_t*)p + at) = out;
  } else {
    *(f4*)((float*)p + at) = f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
    *(f4*)((float*)p + at + 4) = f4{(float)x[4], (float)x[5], (float)x[6], (float)x[7]};
  }
}

}  // namespace

// blockIdx.x: 4 wavefronts' (group, kv head), kv heads fastest.
template <int HD, int TYPE>
__global__ __launch_bounds__(256, 4) void kivi_read_kernel(KiviGeo g, ReadArgs a) {
  constexpr int CH = HD / 8;             // lanes of a token
  constexpr int STEP = 64 / CH;          // tokens at a time
  constexpr int N = kGroup / STEP;       // tokens of a lane
  const int lane = threadIdx.x & 63;
  const int unit = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int h = unit % g.nkv, want = unit / g.nkv;
  // The sequence of the wanted 32, which of its 32s it is, and the rows of the sequences before.
  // A call's tokens may outnumber 32 bits: those past `total` are dropped.
  int64_t before = 0;
  int b = -1, start = 0, end = 0, group = 0, groups = 0;
  for (int base = 0; base < a.batch && b < 0; base += 64) {
    int s = 0, e = 0;
    if (base + lane < a.batch) {
      e = clamp_len(g, a.ends[base + lane]);
      s = a.starts[base + lane];
      s = s < 0 ? 0 : s > e ? e : s;
    }
    const int n = e > s ? (e + kGroup - 1) / kGroup - s / kGroup : 0;
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
  int old, residual;
  decode_window(g, end, &old, &residual);
  const int t0 = start / kGroup * kGroup + group * kGroup;
  const int ch = lane % CH * 8, r0 = lane / CH;
  // the rows of this lane's tokens, and whether they are wanted
  auto row = [&](int i) { return before + t0 + r0 + i * STEP - start; };
  auto there = [&](int i) {
    const int t = t0 + r0 + i * STEP;
    return t >= start && t < end && row(i) < a.total;
  };
  if (t0 >= old) {
    const int64_t base = (((int64_t)b * g.nkv + h) * g.rs + (t0 - old) + r0) * HD + ch;
    u4 k[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (there(i)) {
        k[i] = *(const u4*)(a.pool.k_scr + base + i * STEP * HD);
        v[i] = *(const u4*)(a.pool.v_scr + base + i * STEP * HD);
      }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (there(i)) {
        const int64_t at = (row(i) * g.nkv + h) * HD + ch;
        store8<TYPE>(a.k, at, k[i]);
        store8<TYPE>(a.v, at, v[i]);
      }
    return;
  }
  // A group lies in one page or two; its scales of K in the first, without which its tokens of the
  // second are not there either.
  const int32_t* table = a.tables + (int64_t)b * g.max_pages + t0 / g.page;
  int page[2];
  bool ok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    page[i] = table[g.page == 16 ? i : 0];
    ok[i] = page[i] >= 0 && page[i] < g.num_pages;
    page[i] = ok[i] ? page[i] : 0;
    ok[i] &= ok[0];
  }
  h2 ks[4], kz[4];
  {
    const int64_t at = ((int64_t)page[0] * g.nkv + h) * HD + ch;
    const u4 s = *(const u4*)(a.pool.k_scale + at), z = *(const u4*)(a.pool.k_zero + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ks[i] = pair(s[i]);
      kz[i] = pair(z[i]);
    }
  }
  uint32_t kc[N], vc[N], vs[N], vz[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = r0 + i * STEP;
    const int64_t at = ((int64_t)page[r >> 4] * g.nkv + h) * g.page + (r & (g.page - 1));
    kc[i] = *(const uint32_t*)(a.pool.k_code + at * (HD / 2) + ch / 2);
    vc[i] = *(const uint32_t*)(a.pool.v_code + at * (HD / 2) + ch / 2);
    vs[i] = a.pool.v_scale[at * (HD / 32) + ch / 32];
    vz[i] = a.pool.v_zero[at * (HD / 32) + ch / 32];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!there(i)) continue;
    const bool here = ok[(r0 + i * STEP) >> 4];
    const h2 s = pair(vs[i] | vs[i] << 16), z = pair(here ? vz[i] | vz[i] << 16 : 0x7e007e00u);
    const h2 s4[4] = {s, s, s, s}, z4[4] = {z, z, z, z};
    h2 kk[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) kk[c] = here ? kz[c] : pair(0x7e007e00u);
    const int64_t at = (row(i) * g.nkv + h) * HD + ch;
    store8<TYPE>(a.k, at, kc[i], ks, kk);
    store8<TYPE>(a.v, at, vc[i], s4, z4);
  }
}

template <int HD>
static void read_kernels(const KiviGeo& g, const ReadArgs& a, int type, hipStream_t s) {
  // a sequence's tokens touch at most one group of 32 more than a 32nd of them, begun ones counted
  const unsigned units = (unsigned)g.nkv * (a.total / kGroup + 2 * a.batch);
  const dim3 grid((units + 3) / 4), block(256);
  if (type == kFp16) hipLaunchKernelGGL((kivi_read_kernel<HD, kFp16>), grid, block, 0, s, g, a);
  else if (type == kBf16) hipLaunchKernelGGL((kivi_read_kernel<HD, kBf16>), grid, block, 0, s, g, a);
  else hipLaunchKernelGGL((kivi_read_kernel<HD, kFp32>), grid, block, 0, s, g, a);
}

hipError_t launch_kivi_read(const KiviGeo& g, const KiviPool& p, const int32_t* starts,
                            const int32_t* ends, const int32_t* tables, int batch, int total, void* k,
                            void* v, int type, hipStream_t s) {
  const ReadArgs a = {p, starts, ends, tables, k, v, batch, total};
  if (g.hd == 128) read_kernels<128>(g, a, type, s);
  else read_kernels<64>(g, a, type, s);
  return hipGetLastError();
}

}  // namespace jacq
