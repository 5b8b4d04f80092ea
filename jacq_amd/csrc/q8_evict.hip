// q8_evict.hip -- which blocks of a sequence leave the cache.
//
// One workgroup per sequence, K consecutive entries of the row a thread, all in
// registers: what is read is read before anything is written, so the outputs
// may be the inputs.  The weights become unsigned keys in their order; four
// histogram passes of 8 bits find the key of the lightest kept block and how
// many blocks of that key stay (the earlier ones).  Every wavefront looks
// through a histogram by itself, so a pass costs one barrier; two prefix sums
// then give every entry its place.  What it takes is that chain, not bytes:
// 64 rows of 2048 entries 9.1 us, 1.3 MB.
#include "q8_common.h"

namespace jacq {
namespace q8 {

// Order of weights as unsigned numbers; NaN lightest, -0 as 0.
__device__ inline uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return u >> 31 ? ~u : u | 0x80000000u;  // of a number never 0
}

struct EvictArgs {
  const float* w;
  const int32_t* lens;
  const int32_t* tables;
  int32_t* tables_out;
  int32_t* lens_out;
  float* w_out;
  int32_t* evicted;
  int batch, keep, sink, recent;
};

// Sum over the threads before this one.  `sums` is of its own for every call.
template <int WAVES>
__device__ inline int sum_before(int x, int* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inc = wave_prefix(x, Sum());
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  int sum = inc - x;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) sum += i < wave ? sums[i] : 0;
  return sum;
}

template <int THREADS, int K>
__global__ __launch_bounds__(THREADS) void q8_evict_kernel(Geo g, EvictArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ uint32_t hist[4][256];
  __shared__ int sums[2][WAVES];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int64_t row = (int64_t)b * g.max_pages;
  const float* w = a.w + row;
  const int32_t* table = a.tables + row;
  float* w_out = a.w_out + row;
  int32_t* table_out = a.tables_out + row;
  const int raw = a.lens[b];
  float x[K];
  int32_t entry[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {  // with the length's load, not after it, and without branches
    const int i = tid * K + k, at = i < g.max_pages ? i : g.max_pages - 1;
    x[k] = w[at];
    entry[k] = table[at];
  }
  const int len = clamp_len(g, raw), full = len >> g.page_log2;
  const int drop = full > a.keep ? full - a.keep : 0;
  for (int i = tid; i < 4 * 256; i += THREADS) (&hist[0][0])[i] = 0;
  if (drop == 0) {  // of all of the workgroup
    if (tid == 0) {
      a.evicted[b] = 0;
      if (a.lens_out != a.lens) a.lens_out[b] = raw;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = tid * K + k;
      if (i < g.max_pages) {
        if (table_out != table) table_out[i] = entry[k];
        if (w_out != w) w_out[i] = x[k];
      }
    }
    return;
  }
  const int lo = a.sink, hi = full - a.recent;  // candidates
  const int stay = a.keep - a.sink - a.recent;  // of them kept, fewer than there are
  __syncthreads();
  uint32_t found = 0, mask = 0;
  int want = stay;
  if (stay > 0) {
#pragma unroll 1  // few workgroups run this once: its code has to be fetched, so it is short
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = tid * K + k;
        const uint32_t key = weight_key(x[k]);
        if (i >= lo && i < hi && (key & mask) == found)
          atomicAdd(&hist[pass][key >> shift & 255], 1u);
      }
      __syncthreads();
      // lane: 4 bins, from the heaviest down
      const int top = 255 - 4 * lane;
      const int c0 = hist[pass][top], c1 = hist[pass][top - 1], c2 = hist[pass][top - 2],
                c3 = hist[pass][top - 3];
      const int own = c0 + c1 + c2 + c3, inc = wave_prefix(own, Sum());
      int above = inc - own, bin = top;
      const uint64_t here = __ballot(above < want && inc >= want);  // one lane
      if (above + c0 < want) {
        above += c0;
        --bin;
        if (above + c1 < want) {
          above += c1;
          --bin;
          if (above + c2 < want) {
            above += c2;
            --bin;
          }
        }
      }
      const int l = __builtin_ctzll(here);
      found |= (uint32_t)__builtin_amdgcn_readlane(bin, l) << shift;
      mask |= 255u << shift;
      want -= __builtin_amdgcn_readlane(above, l);
    }
  }
  // Heavier than `found`: kept; equal: the first `want` of them.
  int ties = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = tid * K + k;
    ties += i >= lo && i < hi && stay > 0 && weight_key(x[k]) == found;
  }
  int equal = sum_before<WAVES>(ties, sums[0]);
  uint32_t keeps = 0;  // bit k
  static_assert(K <= 32, "a bit per entry");
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = tid * K + k;
    const uint32_t key = weight_key(x[k]);
    const bool cand = i >= lo && i < hi, tie = cand && stay > 0 && key == found;
    const bool keep = i < full && (!cand || (stay > 0 && key > found) || (tie && equal < want));
    equal += tie;
    keeps |= (uint32_t)keep << k;
  }
  int kept = sum_before<WAVES>(__popc(keeps), sums[1]);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = tid * K + k;
    if (i < full) {
      const bool keep = keeps >> k & 1;
      table_out[keep ? kept : a.keep + i - kept] = entry[k];
      if (keep) w_out[kept] = x[k];
      kept += keep;
    } else if (i < g.max_pages) {
      if (table_out != table) table_out[i] = entry[k];
      if (i == full) w_out[a.keep] = x[k];  // the block in progress keeps its weight
    }
    // behind the kept blocks and that one nothing has a weight
    if (i < g.max_pages && (i > a.keep || (i == a.keep && full == g.max_pages))) w_out[i] = 0.0f;
  }
  if (tid == 0) {
    a.evicted[b] = drop;
    a.lens_out[b] = len - (drop << g.page_log2);
  }
}

template <int THREADS, int K>
static void evict(const Geo& g, const EvictArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((q8_evict_kernel<THREADS, K>), dim3(a.batch), dim3(THREADS), 0, s, g, a);
}

hipError_t launch_evict(const Geo& g, const float* w, const int32_t* lens, const int32_t* tables,
                        int batch, int keep, int sink, int recent, int32_t* tables_out,
                        int32_t* lens_out, float* w_out, int32_t* evicted, hipStream_t s) {
  const EvictArgs a = {w,     lens, tables, tables_out, lens_out, w_out, evicted,
                       batch, keep, sink,   recent};
  // the fewest wavefronts that hold the row: a barrier of 4 is cheaper than one of 16
  static_assert(JACQ_Q8_MAX_PAGES_PER_SEQ == 1024 * 16, "the longest row");
  if (g.max_pages <= 1024) evict<256, 4>(g, a, s);
  else if (g.max_pages <= 2048) evict<256, 8>(g, a, s);
  else if (g.max_pages <= 8192) evict<1024, 8>(g, a, s);
  else evict<1024, 16>(g, a, s);
  return hipGetLastError();
}

}  // namespace q8
}  // namespace jacq
