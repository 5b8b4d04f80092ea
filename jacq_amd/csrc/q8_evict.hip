// q8_evict.hip -- which blocks of a sequence leave the cache.
//
// One workgroup per sequence.  The weights become unsigned keys in their order;
// four histogram passes over 8 bits each find the key of the lightest kept block
// and how many blocks of that key stay (the earlier ones); one more pass deals
// the row's entries out, kept and evicted, each in order, by a prefix sum over
// the workgroup.  What it takes is the chain of passes, not bytes.
#include "q8_common.h"

namespace jacq {
namespace q8 {

constexpr int kThreads = 1024;
constexpr int kInRegs = 4;  // entries of a thread that stay in registers over the passes

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

// Exclusive sum over the workgroup of two counts of at most 2^15 each, packed.
__device__ inline uint32_t prefix(uint32_t x, uint32_t* sums, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const uint32_t s = sums[i];
    before += i < wave ? s : 0;
    all += s;
  }
  __syncthreads();
  *total = all;
  return before + inc - x;
}

__global__ __launch_bounds__(kThreads) void q8_evict_kernel(Geo g, EvictArgs a) {
  extern __shared__ int32_t gone[];  // evicted entries, in order: TABLES_OUT may be the input
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sums[kThreads / 64];
  __shared__ uint32_t pick[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int64_t row = (int64_t)b * g.max_pages;
  const float* w = a.w + row;
  const int32_t* table = a.tables + row;
  const int len = clamp_len(g, a.lens[b]);
  const int full = len >> g.page_log2;
  const int drop = full > a.keep ? full - a.keep : 0;
  if (tid == 0) a.evicted[b] = drop;
  if (drop == 0) {
    if (tid == 0 && a.lens_out != a.lens) a.lens_out[b] = a.lens[b];
    for (int i = tid; i < g.max_pages; i += kThreads) {
      if (a.tables_out != a.tables) a.tables_out[row + i] = table[i];
      if (a.w_out != a.w) a.w_out[row + i] = w[i];
    }
    return;
  }
  const int lo = a.sink, hi = full - a.recent;  // candidates
  const int stay = a.keep - a.sink - a.recent;  // of them kept, less than there are
  uint32_t key[kInRegs];
#pragma unroll
  for (int k = 0; k < kInRegs; ++k) {
    const int i = lo + tid + k * kThreads;
    key[k] = i < hi ? weight_key(w[i]) : 0;
  }
  // The key of the stay-th heaviest candidate, 8 bits at a time from the top.
  uint32_t found = 0, mask = 0;
  int want = stay;
  if (stay > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kInRegs; ++k) {
        const int i = lo + tid + k * kThreads;
        if (i < hi && (key[k] & mask) == found) atomicAdd(&hist[key[k] >> shift & 255], 1u);
      }
      for (int i = lo + tid + kInRegs * kThreads; i < hi; i += kThreads) {
        const uint32_t x = weight_key(w[i]);
        if ((x & mask) == found) atomicAdd(&hist[x >> shift & 255], 1u);
      }
      __syncthreads();
      if (tid < 64) {  // lane: 4 bins from the heaviest down
        const int top = 255 - 4 * tid;
        const uint32_t c0 = hist[top], c1 = hist[top - 1], c2 = hist[top - 2], c3 = hist[top - 3];
        uint32_t inc = c0 + c1 + c2 + c3;
        const uint32_t own = inc;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t y = __shfl_up(inc, d);
          if (tid >= d) inc += y;
        }
        uint32_t above = inc - own;
        if (above < (uint32_t)want && inc >= (uint32_t)want) {  // one lane
          int bin = top;
          if (above + c0 < (uint32_t)want) { above += c0; --bin;
            if (above + c1 < (uint32_t)want) { above += c1; --bin;
              if (above + c2 < (uint32_t)want) { above += c2; --bin; } } }
          pick[0] = (uint32_t)bin;
          pick[1] = above;
        }
      }
      __syncthreads();
      found |= pick[0] << shift;
      mask |= 255u << shift;
      want -= (int)pick[1];
      __syncthreads();
    }
  }
  // Heavier than `found`: kept; equal: the first `want` of them.  In chunks of kThreads entries,
  // low half of a count: kept so far, high half: equal ones so far.
  int kept = 0, equal = 0;
  for (int base = 0; base < full; base += kThreads) {
    const int i = base + tid;
    const bool in = i < full, cand = in && i >= lo && i < hi;
    const float wi = in ? w[i] : 0.0f;
    const int32_t entry = in ? table[i] : 0;
    const uint32_t x = weight_key(wi);
    const bool tie = cand && stay > 0 && x == found;
    uint32_t total;
    const uint32_t e = prefix(tie ? 1u : 0u, sums, &total);
    const bool keep = in && (!cand || (stay > 0 && x > found) || (tie && equal + (int)e < want));
    equal += (int)total;
    const uint32_t k = prefix(keep ? 1u : 0u, sums, &total);  // all of the chunk is read by now
    if (keep) {
      const int to = kept + (int)k;  // <= i: nothing unread is overwritten
      a.tables_out[row + to] = entry;
      a.w_out[row + to] = wi;
    } else if (in) {
      gone[i - (kept + (int)k)] = entry;
    }
    kept += (int)total;
  }
  const bool open = full < g.max_pages;  // the block in progress keeps its weight
  const float last = open ? w[full] : 0.0f;  // at full > keep, which nothing has overwritten
  __syncthreads();
  if (tid == 0) a.lens_out[b] = len - (drop << g.page_log2);  // all have read the length
  for (int i = tid; i < drop; i += kThreads) a.tables_out[row + a.keep + i] = gone[i];
  if (a.tables_out != a.tables)
    for (int i = full + tid; i < g.max_pages; i += kThreads) a.tables_out[row + i] = table[i];
  for (int i = a.keep + tid; i < g.max_pages; i += kThreads)
    a.w_out[row + i] = open && i == a.keep ? last : 0.0f;
}

hipError_t launch_evict(const Geo& g, const float* w, const int32_t* lens, const int32_t* tables,
                        int batch, int keep, int sink, int recent, int32_t* tables_out,
                        int32_t* lens_out, float* w_out, int32_t* evicted, hipStream_t s) {
  const EvictArgs a = {w,       lens,  tables, tables_out, lens_out, w_out, evicted,
                       batch,   keep,  sink,   recent};
  const int most = g.max_pages > keep ? g.max_pages - keep : 0;
  if (most > 16384 - 512) {  // past 64 KiB a kernel asks for its LDS
    const hipError_t e = hipFuncSetAttribute((const void*)q8_evict_kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, most * 4);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(q8_evict_kernel, dim3(batch), dim3(kThreads), (size_t)most * 4, s, g, a);
  return hipGetLastError();
}

}  // namespace q8
}  // namespace jacq
