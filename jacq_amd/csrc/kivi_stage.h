// kivi_stage.h -- the int4 cache's groups on their way to the matrix cores: LDS DMA of a group's codes,
// scales and zeros, and which tokens an operand's rows are.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

#include <type_traits>
#include <utility>

#include "kivi_common.h"

namespace jacq {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int HD, int P>
struct Cfg {
  static constexpr int KS = HD / 32;       // k-steps of the QK^T product
  static constexpr int CPL = HD / 16;      // V channels per lane = PV N-tiles
  static constexpr int HDP = HD / 2;       // packed bytes per token row
  static constexpr int HDG = HD / kGroup;  // V scale groups per token
  static constexpr int KCB = HD / 8;       // K code bytes per lane per token
  static constexpr int PPG = kGroup / P;   // pages per 32-token group
  typedef typename std::conditional<HD == 128, u32x4, u32x2>::type kvec;
  typedef typename std::conditional<HD == 128, u32x2, uint32_t>::type pvec;
};

// Token <-> MFMA position maps of a quantised group.  The QK^T A operand
// row c of tile tt holds token tok_k(tt, c); the PV K index 8j + e (lane
// quarter j, element e) is token tok_v(j, e).  They agree -- S^T row 4j + i of
// tile tt lands in lane quarter j, element 4tt + i -- so P leaves the softmax
// already in PV A-operand order.  Within a 32-lane half the 16 rows a V read
// touches alternate in parity, which keeps ds_read_b32 free of bank conflicts
// on the row-major LDS image of the codes.
__device__ constexpr int tok_k(int tt, int c) {
  return 8 * tt + 2 * (c & 3) + ((c >> 2) & 1) + 16 * (c >> 3);
}
__device__ constexpr int tok_v(int j, int e) { return 2 * e + (j & 1) + 16 * (j >> 1); }

// One quantised 32-token group of one kv head in LDS.  Codes keep the cache's
// row-major order (token rows of HD/2 bytes); scales and zeros arrive as
//   s[0, 2HD)        K scale of channel d at 2d
//   s[2HD, 4HD)      K zero
//   s[4HD, ..)       V scale of (token t, group g) at 2(t*HDG + g), then V zero.
// Everything comes by LDS DMA with 16 bytes per lane (global_load_lds_dwordx4
// puts lane i's bytes at 16i): an LDS DMA costs about the same issue time
// whatever its width, so a group is 2 * 32*HD/2 / 1024 + 1 of them.  The DMAs
// are issued from inline asm and waited for with explicit vmcnt counts: a
// ring of stages keeps S - 1 groups in flight while one is computed.

template <int HD>
constexpr int code_dmas() {  // 1 KiB DMAs per K or V code block
  return 32 * HD / 2 / 1024;
}

// vector memory instructions one stage issues (vmcnt units)
template <int HD>
constexpr int stage_loads() {
  return 2 * code_dmas<HD>() + 1;
}

// Per-segment DMA sources.  Codes: wave-uniform bases (kv head folded in);
// scales: the lane's own 16-byte word of page 0 and the page stride of its
// array (K scales live once per group, in its first page).
struct StageBases {
  uint64_t kc, vc;     // k_code / v_code + head offset (uniform)
  uint32_t code_page;  // bytes per physical page of K or V codes (all kv heads)
  uint64_t sc;         // lane's scale / zero source in page 0
  uint32_t sc_page;    // lane's page stride in bytes
  bool sc_p1;          // lane's word lies in the group's second page
  bool sc_on;          // lane takes part in the scale DMA
};

template <int HD, int P, class A>
__device__ inline StageBases stage_bases(const A& a, int nkv, int h, int lane) {
  using C = Cfg<HD, P>;
  asm volatile("" : "+v"(lane));  // per segment, not hoisted into the whole run
  constexpr int KL = HD / 8;          // lanes per K scale (or zero) row
  constexpr int VL = 4 * C::HDG;      // lanes per V scale (or zero) block of 32 tokens
  StageBases sb;
  sb.code_page = (uint32_t)(nkv * P * C::HDP);
  sb.kc = (uint64_t)(a.k_code + (int64_t)h * P * C::HDP);
  sb.vc = (uint64_t)(a.v_code + (int64_t)h * P * C::HDP);
  sb.sc_on = lane < 2 * KL + 2 * VL;
  sb.sc_p1 = false;
  if (lane < 2 * KL) {
    const uint16_t* arr = lane < KL ? a.k_scale : a.k_zero;
    sb.sc = (uint64_t)(arr + (int64_t)h * HD + 8 * (lane % KL));
    sb.sc_page = (uint32_t)(nkv * HD * 2);
  } else {
    const int l = (lane - 2 * KL) % VL;
    const uint16_t* arr = lane < 2 * KL + VL ? a.v_scale : a.v_zero;
    const int t = 8 * l / C::HDG;  // first token of the lane's word
    sb.sc_p1 = t >= P;
    sb.sc = (uint64_t)(arr + ((int64_t)h * P + t % P) * C::HDG);
    sb.sc_page = (uint32_t)(nkv * P * C::HDG * 2);
  }
  return sb;
}

__device__ inline uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// LDS DMA of SZ bytes per lane from addr + OFF to LDS byte dst + lane * max(SZ, 4),
// non-temporal: every cache byte is read once per decode step, and streaming
// it past the caches sustains a markedly higher HBM read rate.
// The instruction's immediate offset moves the LDS address as well as the
// global one, so M0 gets dst - OFF.  M0 is set inside the same asm statement,
// so nothing the compiler keeps in M0 is live across it.  An LDS DMA must not
// read M0 in the instruction right after the SALU write of it (the GFX9
// M0 / LDS-DMA hazard: one wait state); the compiler's hazard recognizer does
// not look inside asm, so the s_nop is written here.
// COH: device-scope load (sc1) instead of the non-temporal hint -- for data
// another wavefront of the same launch stored with device-scope stores (the
// fused step's age-outs), which a non-temporal load could find stale in this
// XCD's L2.
template <int SZ, int OFF, bool COH = false>
__device__ inline void dma(uint64_t addr, uint32_t dst) {
  static_assert(OFF >= 0 && OFF < 4096, "global immediate offset range");
  const uint32_t m0 = dst - OFF;
  if constexpr (COH) {
    static_assert(SZ == 16, "device-scope LDS DMA: 16 bytes per lane");
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2 sc1"
                 :: "s"(m0), "v"(addr), "n"(OFF) : "memory", "m0");
  } else if constexpr (SZ == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2 nt"
                 :: "s"(m0), "v"(addr), "n"(OFF) : "memory", "m0");
  else if constexpr (SZ == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off offset:%2 nt"
                 :: "s"(m0), "v"(addr), "n"(OFF) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off offset:%2 nt"
                 :: "s"(m0), "v"(addr), "n"(OFF) : "memory", "m0");
}

// The same with a wave-uniform 64-bit base in SGPRs and a 32-bit lane offset.
template <int OFF, bool COH = false>
__device__ inline void dma16s(uint64_t sbase, uint32_t voff, uint32_t dst) {
  static_assert(OFF >= 0 && OFF < 4096, "global immediate offset range");
  const uint32_t m0 = dst - OFF;
  if constexpr (COH)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3 sc1"
                 :: "s"(m0), "v"(voff), "s"(sbase), "n"(OFF) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3 nt"
                 :: "s"(m0), "v"(voff), "s"(sbase), "n"(OFF) : "memory", "m0");
}

template <int N>
__device__ inline void wait_vm() {  // at most N vector memory ops outstanding
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

template <class F, int... I>
__device__ inline void static_for_impl(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ inline void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Issue the DMAs of one group whose tokens 0..P-1 sit in page p0 and the
// rest (page size 16) in p1.
template <int HD, int P, bool COH = false, class Buf>
__device__ inline void load_stage(Buf* buf, const StageBases& sb, uint32_t p0,
                                  uint32_t p1, int lane) {
  const uint32_t base = lds_addr(buf);
  const uint32_t kd = base + (uint32_t)offsetof(Buf, k);
  const uint32_t vd = base + (uint32_t)offsetof(Buf, v);
  const uint32_t lo = 16u * (uint32_t)lane;
  if constexpr (HD == 128) {
    // 1 KiB = 16 token rows per DMA: rows 0-15 and 16-31
    const uint64_t o0 = (uint64_t)p0 * sb.code_page;
    const uint64_t o1 = P == 16 ? (uint64_t)p1 * sb.code_page : o0 + 1024;
    dma16s<0, COH>(sb.kc + o0, lo, kd);
    dma16s<0, COH>(sb.kc + o1, lo, kd + 1024);
    dma16s<0, COH>(sb.vc + o0, lo, vd);
    dma16s<0, COH>(sb.vc + o1, lo, vd + 1024);
  } else if constexpr (P == 32) {
    const uint64_t o0 = (uint64_t)p0 * sb.code_page;
    dma16s<0, COH>(sb.kc + o0, lo, kd);
    dma16s<0, COH>(sb.vc + o0, lo, vd);
  } else {
    // one DMA spans both pages: lanes 0-31 rows 0-15 of p0, lanes 32-63 of p1
    const uint64_t o = (uint64_t)(lane < 32 ? p0 : p1) * sb.code_page + (lo & 511u);
    dma<16, 0, COH>(sb.kc + o, kd);
    dma<16, 0, COH>(sb.vc + o, vd);
  }
  const uint32_t sd = base + (uint32_t)offsetof(Buf, s);
  const uint64_t sa = sb.sc + (uint64_t)(sb.sc_p1 ? p1 : p0) * sb.sc_page;
  if (sb.sc_on) dma<16, 0, COH>(sa, sd);
}

// IEEE maximum (llvm.maximum): lowers to v_maximum3_f32 without the
// canonicalising moves that fmaxf needs in IEEE mode.
__device__ inline float max3f(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
__device__ inline float max2f(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// max with lane l ^ 16 / l ^ 32 by v_permlane16_swap / v_permlane32_swap
// (all VALU, no LDS round trip).  Both operands start as x; after the swap one
// holds this lane's row value and the other the partner row's.  Written as
// asm with both operands read-write: the compiler's lowering of the builtin
// reads the first result register for both results.  The s_nop gives the
// VALU write of x the wait states the swap needs.
__device__ inline float max_xor16(float x) {
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return max2f(a, b);
}
__device__ inline float max_xor32(float x) {
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return max2f(a, b);
}

}  // namespace jacq
