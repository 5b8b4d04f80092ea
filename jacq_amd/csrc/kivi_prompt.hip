// kivi_prompt.hip -- attention of prompts over the int4 cache.
//
// Every row tile of a kv head takes in the same tokens, so they become fp16 once: kivi_lay_kernel writes
// tiles of 64 tokens, K [64][HD] and V^T [HD][64], to the workspace as the LDS will hold them, and
// kivi_prompt_kernel copies them by LDS DMA, without a register or a vector instruction in between.
//
// A workgroup has 128 query rows of one kv head (row = query token x head of the group), 32 for each of 4
// wavefronts, and goes through the tiles that any of its rows sees, or through one of several slices of
// them.  S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_f16; a lane's column is a query row, so its
// maximum, sum and rescaling are the lane's own (and its partner's, 32 lanes on), and the order in which
// K's rows enter makes P the next operand as it stands.
//
// HD 128 is bound by the LDS (32 rows take in 32 KB a tile) and by the clock, which falls to 1.7 GHz under
// matrix instructions, HD 64 by vector instructions (145 a tile, 16 matrix ones).  A prompt of 8191 tokens,
// 40/8 heads of 128: 667 to 690 us, 640 of them this kernel's, 1073 TFLOP/s of the 1202 that a large library
// product reaches; laying its tiles takes 14 us.  Six of 1448 to 7790, 14/2 heads of 64, window 1024: 155 us,
// 620 TFLOP/s.  The softmax between the next tile's products, in the order of the source, was slower (736
// and 176 us): three or four wavefronts a SIMD do it by themselves.
#include "kivi_attend.h"
#include "kivi_stage.h"

namespace jacq {

namespace {

constexpr int kPromptWaves = 4;
// A slice's share of the tiles is such that as many equal slices would fill the CUs kRounds times.  Slices
// even the lengths out, but their parts are written and joined.  us, with 0.35, 0.5, 0.7, 1, 2 and 3: 511
// queries of each of 4 sequences of 6834 to 14251 tokens, 32/8 heads of 128, 433, 425, 408, 424, 433 and 438;
// 333 of each of 8 of 1451 to 5722 245, 245, 236, 245, 253 and 250.  24 calls of random sizes, in geometric
// mean, with 0.5, 0.6, 0.7 and 0.85: 73.4, 72.6, 72.8 and 73.6.
constexpr float kRounds = 0.7f;
static_assert(kPrefillRows == 32 * kPromptWaves, "32 rows a wavefront");

// Where chunk c (8 values) of a row of an image lies, so that 16 rows' same chunk covers all banks.
template <int HD>
__device__ inline int k_chunk(int row, int c) {
  return HD == 128 ? c ^ (row & 15) : c ^ (row >> 1 & 7);
}
__device__ inline int v_chunk(int d, int c) { return c ^ (d >> 1 & 7); }

template <int HD>
struct Image {
  uint16_t k[kTile][HD];
  uint16_t v[HD][kTile];
};

// The kernel's own copies of 16 bytes a lane from base + lane offset to LDS dst + 16 lane; tiles are read
// by many workgroups, so they may stay in the caches.
template <int OFF>
__device__ inline void copy16(uint64_t base, uint32_t lane16, uint32_t dst) {
  static_assert(OFF >= 0 && OFF < 4096, "immediate offset");
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
               :: "s"(dst), "v"(lane16), "s"(base), "n"(OFF) : "memory", "m0");
}

// Where a sequence's images are: those of kv head h from first + h units on, if they are of this pass.
// A sequence without tokens has none, and is the first pass's: its place, the next one's first image, may be
// behind the last pass.
__device__ inline bool images_of(const KiviGeo& g, const KiviAttendArgs& a, int b, int pass, int units,
                                 int h, int64_t* at) {
  if (units == 0) {
    *at = 0;
    return pass == 0;
  }
  const int slot = uniform(a.slots[b]);
  if (slot / a.per_pass != pass) return false;
  *at = (int64_t)(slot % a.per_pass) * g.nkv + (int64_t)h * units;
  return true;
}

// A sequence's images, and the tiles that its row tiles go through.
__device__ inline int images_and_work(const KiviGeo& g, const KiviAttendArgs& a, int b, float& work) {
  int q0, m, all;
  queries_of(a, b, &q0, &m, &all);
  work = 0.0f;
  if (m == 0) return 0;
  const KiviTiles tiles(g, a, clamp_len(g, a.lens[b]), a.causal ? clamp_len(g, a.lens[b]) - all
                                                                : clamp_len(g, a.lens[b]) - 1);
  work = (float)((m * g.gqa + kPrefillRows - 1) / kPrefillRows) * row_tiles_units(a, tiles, m, all);
  return tiles.units;
}

__device__ inline float slice_share(const KiviGeo& g, const KiviAttendArgs& a, float work) {
  const float share = work * (float)g.nkv / (kRounds * (float)(prompt_groups(g.hd) * a.cus));
  return share > (float)kSliceUnits ? share : (float)kSliceUnits;
}

}  // namespace

// The first image of every sequence, and a slice's share of the tiles that row tiles go through, of more
// than kCounted sequences (kivi_lay_kernel finds those of fewer by itself, a launch and 2 to 4 us less).  Offsets
// that go back can give more sequences queries than there are queries, and more images than the workspace
// has room for: those behind a.limit are left out.  One workgroup.
__global__ __launch_bounds__(1024) void kivi_slots_kernel(KiviGeo g, KiviAttendArgs a) {
  __shared__ int sums[2][16];
  __shared__ float work[16];
  __shared__ int out;  // the first image that is left out
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int before = 0;
  if (tid == 0) out = INT32_MAX;
  float w = 0.0f;
  for (int base = 0, turn = 0; base < a.batch; base += 1024, turn ^= 1) {
    const int b = base + tid;
    float own = 0.0f;
    const int units = b < a.batch ? images_and_work(g, a, b, own) : 0;
    w += own;
    const int inc = wave_prefix(units, Sum());
    if (lane == 63) sums[turn][wave] = inc;
    __syncthreads();  // the other turn's sums have been read by all
    int here = before + inc - units;
    for (int i = 0; i < 16; ++i) {
      here += i < wave ? sums[turn][i] : 0;
      before += sums[turn][i];
    }
    if (b < a.batch) {
      const bool fits = here <= a.limit - units;
      a.slots[b] = fits ? here : INT32_MAX;
      if (!fits) atomicMin(&out, here);
    }
  }
  w = __int_as_float(lane63(wave_prefix(__float_as_int(w), SumF())));
  if (lane == 0) work[wave] = w;
  __syncthreads();
  if (tid == 0) {
    a.slots[a.batch] = before < out ? before : out;
    w = 0.0f;
    for (int i = 0; i < 16; ++i) w += work[i];
    a.slots[a.batch + 1] = __float_as_int(slice_share(g, a, w));
  }
}

// The images of a pass, one at a time (blockIdx.y: kv head).  HD threads have V, a chunk of 8 channels of 8
// tokens each, HD have K, a chunk of 8 channels of 8 tokens of a group each.  Through the LDS, so that
// whole lines are written.
template <int HD, int P>
__global__ __launch_bounds__(2 * HD) void kivi_lay_kernel(KiviGeo g, KiviAttendArgs a, int pass) {
  constexpr int CH = HD / 8;  // chunks of a row
  __shared__ __align__(16) Image<HD> image;
  __shared__ uint32_t bad[kTile / 8];
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y;
  const bool is_v = uniform(tid / HD) == 0;
  const int chunk = tid % HD % CH, part = tid % HD / CH;  // part: V: 8 tokens; K: 4 of a group's rows
  const int64_t begin = (int64_t)pass * a.per_pass;
  const bool few = a.batch <= kCounted;
  int mine = 0, total;  // few: the first image of the lane's sequence
  if (few) {
    float w = 0.0f;
    const int units = lane < a.batch ? images_and_work(g, a, lane, w) : 0;
    const int inc = wave_prefix(units, Sum());
    const bool fits = inc <= a.limit;
    mine = fits ? inc - units : INT32_MAX;
    // the images before the first one that does not fit
    const uint64_t not_ = __ballot(!fits);
    total = not_ ? __builtin_amdgcn_readlane(inc - units, __builtin_ctzll(not_)) : lane63(inc);
    w = __int_as_float(lane63(wave_prefix(__float_as_int(w), SumF())));
    if (pass == 0 && blockIdx.x == 0 && h == 0 && tid < 64) {  // for the kernels behind this one
      if (lane < a.batch) a.slots[lane] = mine;
      if (lane == 0) {
        a.slots[a.batch] = total;
        a.slots[a.batch + 1] = __float_as_int(slice_share(g, a, w));
      }
    }
  } else {
    total = uniform(a.slots[a.batch]);
  }
  // up to the first sequence of the next pass
  int b = 0;
  for (int64_t slot = begin + blockIdx.x;; slot += gridDim.x) {
    if (slot >= total) return;
    // its sequence: the last one whose first image is not behind it (one without images is not the last)
    if (few) {
      b = 63 - __builtin_clzll(__ballot(lane < a.batch && mine <= slot));
    } else {
      int at = 0;
      for (int n = a.batch; n > 1;) {
        const int step = (n + 63) / 64, i = lane * step;
        const uint64_t upto = __ballot(i < n && a.slots[at + (i < n ? i : 0)] <= slot);
        const int skip = (__popcll(upto) - 1) * step;
        at += skip;
        n = step < n - skip ? step : n - skip;
      }
      b = uniform(at);
    }
    const int first = few ? __builtin_amdgcn_readlane(mine, b) : uniform(a.slots[b]);
    if (first / a.per_pass != pass) {
      if (first >= begin) return;  // the next pass's
      continue;                    // the end of the last pass's
    }
    int q0, m, all;
    queries_of(a, b, &q0, &m, &all);
    const int n = clamp_len(g, a.lens[b]);
    const KiviTiles tiles(g, a, n, a.causal ? n - all : n - 1);
    const int unit = (int)(slot - first), t0 = tiles.tile_of(unit) * kTile;
    const int half = part >> 2, g0 = t0 + half * kGroup;  // the group, or the fp16 rows, of this thread
    const bool group = g0 < tiles.old;
    int page[2] = {0, 0};
    bool ok[2] = {true, true};
    if (group) {
      const int32_t* table = a.tables + (int64_t)b * g.max_pages + g0 / P;
#pragma unroll
      for (int i = 0; i < kGroup / P; ++i) {
        page[i] = table[i];
        ok[i] = (uint32_t)page[i] < (uint32_t)g.num_pages;
        page[i] = ok[i] ? page[i] : 0;
      }
      if (P == 32) page[1] = page[0], ok[1] = ok[0];
    }
    const int64_t scratch = (((int64_t)b * g.nkv + h) * g.rs + (g0 - tiles.old)) * HD + chunk * 8;
    if (is_v) {
      const int r0 = (part & 3) * 8;  // first of 8 tokens in the group
      uint32_t mask = 0;
      h2 x[4][8];  // tokens 2 p and 2 p + 1, by channel
      if (group) {
        const int64_t at = ((int64_t)page[r0 >> 4] * g.nkv + h) * P + (r0 & (P - 1));
        const uint8_t* code = a.pool.v_code + at * (HD / 2) + chunk * 4;
        const uint16_t* sp = a.pool.v_scale + at * (HD / 32) + chunk / 4;
        const uint16_t* zp = a.pool.v_zero + at * (HD / 32) + chunk / 4;
        uint32_t w[8], s[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = *(const uint32_t*)(code + e * (HD / 2));
          s[e] = sp[e * (HD / 32)];
          z[e] = zp[e * (HD / 32)];
        }
        // a group's scales of K are in its first page
        if (!ok[0] || !ok[r0 >> 4]) mask = 255;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!holds(h2f_((uint16_t)s[e]), h2f_((uint16_t)z[e]))) mask |= 1u << e;
          if (mask >> e & 1) s[e] = z[e] = 0;
        }
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            h2 y[4];
            values8x2(w[2 * p], w[2 * p + 1], odd, pair(s[2 * p] | s[2 * p + 1] << 16),
                      pair(z[2 * p] | z[2 * p + 1] << 16), y);
#pragma unroll
            for (int c = 0; c < 4; ++c) x[p][2 * c + odd] = y[c];
          }
      } else {
        u4 row[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          row[e] = g0 + r0 + e < n ? *(const u4*)(a.pool.v_scr + scratch + (r0 + e) * HD) : u4{0, 0, 0, 0};
          const uint32_t most = most_bits(most_bits(row[e].x, row[e].y), most_bits(row[e].z, row[e].w));
          if (either_half(most) >= 0x7c00u) {
            mask |= 1u << e;
            row[e] = u4{0, 0, 0, 0};
          }
        }
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            x[p][2 * c] = pair(__builtin_amdgcn_perm(row[2 * p + 1][c], row[2 * p][c], 0x05040100u));
            x[p][2 * c + 1] = pair(__builtin_amdgcn_perm(row[2 * p + 1][c], row[2 * p][c], 0x07060302u));
          }
      }
      if (tid < kTile / 8) bad[tid] = 0;  // lanes 0 to 7; or-ed into below, by lanes of both wavefronts
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = chunk * 8 + c;
        *(u4*)&image.v[d][v_chunk(d, part) * 8] = u4{bits(x[0][c]), bits(x[1][c]), bits(x[2][c]), bits(x[3][c])};
      }
      __syncthreads();
      if (mask) atomicOr(&bad[part], mask);
    } else {
      const int r0 = part & 3;
      if (group) {
        const int64_t at = ((int64_t)page[0] * g.nkv + h) * HD + chunk * 8;
        const u4 s = *(const u4*)(a.pool.k_scale + at), z = *(const u4*)(a.pool.k_zero + at);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + 4 * i;
          w[i] = *(const uint32_t*)(a.pool.k_code +
                                    (((int64_t)page[r >> 4] * g.nkv + h) * P + (r & (P - 1))) * (HD / 2) +
                                    chunk * 4);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = half * kGroup + r0 + 4 * i;
          *(h8*)&image.k[r][k_chunk<HD>(r, chunk) * 8] = values8(w[i], s, z);
        }
      } else {
        u4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + 4 * i;
          w[i] = g0 + r < n ? *(const u4*)(a.pool.k_scr + scratch + r * HD) : u4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = half * kGroup + r0 + 4 * i;
          *(u4*)&image.k[r][k_chunk<HD>(r, chunk) * 8] = w[i];
        }
      }
      __syncthreads();
    }
    __syncthreads();
    const int64_t at = (int64_t)(first % a.per_pass) * g.nkv + (int64_t)h * tiles.units + unit;
    u4* out = (u4*)(a.images + at * (int64_t)sizeof(Image<HD>));
    for (int i = tid; i < (int)sizeof(Image<HD>) / 16; i += 2 * HD) out[i] = ((const u4*)&image)[i];
    if (tid == 0) {
      uint64_t all_bad = 0;
      for (int i = 0; i < kTile / 8; ++i) all_bad |= (uint64_t)bad[i] << 8 * i;
      a.poison[at] = all_bad;
    }
    __syncthreads();  // the image has been read by all
  }
}

template <int HD>
__global__ __launch_bounds__(64 * kPromptWaves, prompt_groups(HD)) void kivi_prompt_kernel(
    KiviGeo g, KiviAttendArgs a, int pass) {
  constexpr int KS = HD / 16;  // k-steps of S^T
  constexpr int DT = HD / 32;  // channel tiles
  struct Lds {
    uint16_t k[2][kTile][HD];
    uint16_t v[HD][kTile];
  };
  extern __shared__ __align__(16) uint8_t shared_bytes[];
  Lds& lds = *(Lds*)shared_bytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int h = blockIdx.x % g.nkv, slice = blockIdx.y;
  if (pass > 0 && (int64_t)pass * a.per_pass >= uniform(a.slots[a.batch])) return;  // of a wide table's
  const Place place = place_of(g, a, blockIdx.x / g.nkv, g.gqa, kRowsLog2);
  const int b = place.b, q0 = place.q0, n = place.n;
  const int rows = place.m * g.gqa;
  const int rt = (rows + kPrefillRows - 1) / kPrefillRows - 1 - place.at;  // the longest first
  if (rt < 0 || place.at < 0) return;
  // positions: the first query's, then the workgroup's and the wavefront's rows; without an order every
  // row stands at the last token
  const int p0 = n - place.all;
  auto position = [&](int row) { return a.causal ? p0 + row / g.gqa : n - 1; };
  const KiviTiles seq(g, a, n, a.causal ? p0 : n - 1);
  const int slices = uniform(kivi_slices(a, seq, place.m, place.all));
  if (slice >= slices) return;
  int64_t image;
  if (!images_of(g, a, b, pass, seq.units, h, &image)) return;
  const int end_row = rows < (rt + 1) * kPrefillRows ? rows : (rt + 1) * kPrefillRows;
  const int pfirst = uniform(position(rt * kPrefillRows));
  const int plast = uniform(position(end_row - 1));
  const int wr0 = rt * kPrefillRows + wave * 32;
  const int wr1 = wr0 + 32 < rows ? wr0 + 32 : rows;
  const int wfirst = uniform(position(wr0));
  const int wlast = uniform(wr0 < rows ? position(wr1 - 1) : -1);

  const int row = wr0 + n32;
  const bool ok = row < rows;
  const int tok = ok ? row / g.gqa : 0, head = h * g.gqa + row % g.gqa;
  const int pos = ok ? position(row) : -1;
  h8 q[KS];
  float mx = kNegInf, l = 0.0f;
  f16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f16v{};
  float qs;
  {
    const uint16_t* src = a.q + (int64_t)(q0 + tok) * a.q_stride + head * HD + hh * 8;
    u4 raw[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) raw[i] = ok ? *(const u4*)(src + i * 16) : u4{0, 0, 0, 0};
    qs = half_row(raw, a.q_bf16, a.scale, q, [](float x) { return fmaxf(x, other_half(x)); });
  }

  // Tiles: the sinks', the window's up to the last row's position; of them this slice's.
  const KiviTiles own(g, a, n, pfirst);
  const int end = (n + kTile - 1) / kTile;
  int top = plast < 0 ? 0 : (plast >> 6) + 1;
  top = top > end ? end : top;
  const int every = plast < 0 ? 0 : own.ns + (top > own.w0 ? top - own.w0 : 0);
  // every slice's tiles but the last one's are as many: below 2^12 tiles, at most 32 slices
  const int share = slices == 1 ? every : (every + slices - 1) / slices;
  const int from = slice * share;
  const int count = uniform(every - from < share ? every - from : share);
  auto tile_at = [&](int u) { return own.tile_of(from + (u < count ? u : count - 1)); };

  // ---- staging: a wavefront copies its quarter of K's and of V's image ----
  constexpr int PART = kTile * HD * 2 / kPromptWaves;
  const uint32_t lane16 = lane * 16;
  const uint64_t images = (uint64_t)a.images + (uint64_t)image * sizeof(Image<HD>) + wave * PART;
  auto copy = [&](uint64_t src, uint32_t dst) {
    static_for<PART / 1024>([&](auto i) { copy16<1024 * i.value>(src, lane16, dst); });
  };
  // Tiles past the last one are copied as the last one again, and never used.
  auto copy_k = [&](int u) {
    copy(images + (uint64_t)seq.unit_of(tile_at(u)) * sizeof(Image<HD>),
         lds_addr(&lds.k[u & 1][0][0]) + wave * PART);
  };
  auto copy_v = [&](int u) {
    copy(images + (uint64_t)seq.unit_of(tile_at(u)) * sizeof(Image<HD>) + kTile * HD * 2,
         lds_addr(&lds.v[0][0]) + wave * PART);
  };

  // K row of this lane in a tile of 32: the scores of a lane are then tokens 8 hh ... + 7 of either half
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
  // Whether all of the wavefront's rows see all of a tile.
  auto whole = [&](int t0) {
    return t0 + kTile - 1 <= wfirst && (a.window <= 0 || t0 > wlast - a.window || t0 + kTile <= a.sinks);
  };
  auto soften = [&](int u, int t0) {
    const uint64_t poison = *(const __attribute__((address_space(4))) uint64_t*)(uintptr_t)(
        a.poison + image + seq.unit_of(tile_at(u)));
    if (poison) {
      const uint64_t mine = poison >> hh * 8;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s[k / 2][(k & 1) * 8 + i] =
              mine >> (16 * k + i) & 1 ? __builtin_nanf("") : s[k / 2][(k & 1) * 8 + i];
    }
    if (!whole(t0)) {
      // bit j: token t0 + j is seen
      uint64_t see = low_bits(pos + 1 - t0);
      if (a.window > 0) see &= ~low_bits(pos + 1 - a.window - t0) | low_bits(a.sinks - t0);
      see >>= hh * 8;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t bits = (uint32_t)(see >> (16 * k));
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // all ones where it is seen: two instructions each
          const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
          s[k / 2][(k & 1) * 8 + i] = __uint_as_float(
              (__float_as_uint(s[k / 2][(k & 1) * 8 + i]) & keep) | (0xff800000u & ~keep));
        }
      }
    }
    float top = kNegInf;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        top = fmaxf(fmaxf(top, s[k / 2][(k & 1) * 8 + i]), s[k / 2][(k & 1) * 8 + i + 1]);
    top = fmaxf(top, other_half(top)) * qs;
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
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = exp2_(__builtin_fmaf(s[k / 2][(k & 1) * 8 + i], qs, -base));
        l += w;
        p[k][i] = (_Float16)w;
      }
  };
  auto values = [&](int u) {
    const uint16_t* vb = &lds.v[0][0];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const h8 v = *(const h8*)(vb + d * 32 * kTile + vo[k]);
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[k], acc[d], 0, 0, 0);
      }
  };
  auto landed = [&] {  // every wavefront's copies
    wait_vm<0>();
    turn();
  };

  if (count > 0) {
    copy_k(0);
    landed();
    copy_v(0);
    copy_k(1);
    for (int u = 0; u < count; ++u) {
      const int t0 = tile_at(u) * kTile;
      scores(u);
      soften(u, t0);
      landed();     // V of u and K of u + 1; and K of u is done with
      copy_k(u + 2);
      values(u);
      turn();       // V of u is done with
      copy_v(u + 1);
    }
    wait_vm<0>();
  }

  l += other_half(l);
  // the row once more, rather than in registers over the loop
  const int end_lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
  const int out_row = wr0 + (end_lane & 31), hh_ = end_lane >> 5;
  if (out_row >= rows) return;
  const int64_t at = (int64_t)(q0 + out_row / g.gqa) * g.nh + h * g.gqa + out_row % g.gqa;
  if (slices > 1) {  // kivi_prompt_merge_kernel joins the slices
    const int64_t part = (int64_t)slice * a.total_q * g.nh + at;
    if (hh_ == 0) {
      a.part_ml[2 * part] = mx;
      a.part_ml[2 * part + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f4*)(a.part_acc + part * HD + d * 32 + i * 8 + hh_ * 4) =
            f4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    return;
  }
  const float inv = over_sum(l, sees_any(g, a, n, p0, out_row / g.gqa));
  if (a.lse && hh_ == 0) a.lse[at] = l == 0.0f ? kNegInf : (mx + log2_(l)) / kLog2e;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f4 x;
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = bounded(g, acc[d][4 * i + c], l) * inv;
      store4(a, at * HD + d * 32 + i * 8 + hh_ * 4, x);
    }
}

template <int HD>
__global__ __launch_bounds__(256) void kivi_prompt_merge_kernel(KiviGeo g, KiviAttendArgs a) {
  merge_slices<HD>(g, a);
}

template <int HD>
static hipError_t prompt_kernels(const KiviGeo& g, const KiviAttendArgs& a, int passes, int64_t images,
                                 hipStream_t s) {
  constexpr int LDS = (2 * kTile * HD + kTile * HD) * 2;
  if (a.batch > kCounted) hipLaunchKernelGGL(kivi_slots_kernel, dim3(1), dim3(1024), 0, s, g, a);
  const dim3 lay((unsigned)images, g.nkv), grid((unsigned)(a.tiles * g.nkv), a.slices);
  for (int pass = 0; pass < passes; ++pass) {
    if (g.page == 16)
      hipLaunchKernelGGL((kivi_lay_kernel<HD, 16>), lay, dim3(2 * HD), 0, s, g, a, pass);
    else
      hipLaunchKernelGGL((kivi_lay_kernel<HD, 32>), lay, dim3(2 * HD), 0, s, g, a, pass);
    hipLaunchKernelGGL((kivi_prompt_kernel<HD>), grid, dim3(64 * kPromptWaves), LDS, s, g, a, pass);
  }
  if (a.slices > 1)
    hipLaunchKernelGGL((kivi_prompt_merge_kernel<HD>), dim3(a.merges), dim3(256), 0, s, g, a);
  return hipGetLastError();
}

hipError_t launch_attend_prompt(const KiviGeo& g, const KiviAttendArgs& a, int passes, hipStream_t s) {
  // workgroups that lay images: one each where they are few
  const int64_t most = (int64_t)a.batch * ((g.lq + g.residual + kTile - 1) / kTile);
  const int64_t images = most < 2048 ? most : 2048;
  return g.hd == 128 ? prompt_kernels<128>(g, a, passes, images, s)
                     : prompt_kernels<64>(g, a, passes, images, s);
}

}  // namespace jacq
