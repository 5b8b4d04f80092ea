// rotary.hip -- rotary positions of queries and keys: kernel and C ABI (include/jacq_rotary.h).
//
// A thread has V pairs of channels of a token (the same of several heads), and finds their cosines and
// sines itself: the angle is position x frequency as a 64-bit fraction of a turn, of which the product
// modulo 2^64 loses nothing at any position (an fp32 product at position 10^6 is off by 0.06 rad); its
// upper 32 bits give the octant and what is left of it, at most 1/8 turn, where the sine's Taylor polynomial
// ends 2^-29 off ((pi/4)^11 / 11!) and the cosine's 2^-25 ((pi/4)^10 / 10!).  No table is read: of HD 128 the V = 8 angles of a thread are about 250 instructions, for
// heads x 32 bytes in and out.
// Bound by latency where there are few tokens (64 of 48 heads: 4 us, of which an empty launch is most),
// by memory where there are many: 16384 of 48 heads of 128, fp16, in 75 us are 5.4 TB/s.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <string>

#include "attend_common.h"
#include "jacq_rotary.h"

namespace jacq {

namespace {

constexpr int kPairs = JACQ_ROTARY_MAX_DIM / 2;

struct RotaryArgs {
  const void* in[2];   // queries, keys
  void* out[2];
  int64_t in_stride[2], out_stride[2];
  int heads[2], out_type[2];
  const void* positions;
  int tokens, hd, rd, positions64, inverse;
  int parts;           // threads' shares of a token's heads
  float amplitude;
  uint64_t turns[kPairs];
};

// cos and sin of `phase` 2^-64 turns.
__device__ inline void cos_sin(uint64_t phase, float& c, float& s) {
  const uint32_t p = (uint32_t)(phase >> 32);
  const uint32_t quarter = (p + 0x20000000u) >> 30;       // the nearest quarter turn
  const int32_t rest = (int32_t)(p - (quarter << 30));    // in 2^-32 turns, at most an eighth
  const float x = (float)rest * 0x1.921fb6p-30f;          // 2 pi 2^-32
  const float y = x * x;
  const float sn = x + x * y * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.0f / 362880, -1.0f / 5040),
                                                                1.0f / 120), -1.0f / 6);
  const float cs = 1.0f + y * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.0f / 40320, -1.0f / 720),
                                                               1.0f / 24), -0.5f);
  const bool swap = quarter & 1;
  const float a = swap ? sn : cs, b = swap ? cs : sn;
  c = ((quarter + 1) & 2) ? -a : a;  // quarters 1 and 2
  s = quarter & 2 ? -b : b;          // quarters 2 and 3
}

template <int T> struct Element { typedef uint16_t type; };
template <> struct Element<kFp32> { typedef uint32_t type; };

// N values, at most 16 bytes a load.
template <int T, int N>
__device__ inline void load(const void* p, int64_t at, float (&x)[N]) {
  typedef typename Element<T>::type E;
  constexpr int B = N * sizeof(E) < 16 ? N : 16 / sizeof(E);
  struct alignas(B * sizeof(E)) Block { E e[B]; };
#pragma unroll
  for (int i = 0; i < N; i += B) {
    const Block b = *(const Block*)((const E*)p + at + i);
#pragma unroll
    for (int j = 0; j < B; ++j)
      x[i + j] = T == kFp32 ? __uint_as_float(b.e[j])
                 : T == kBf16 ? __uint_as_float((uint32_t)b.e[j] << 16) : h2f_((uint16_t)b.e[j]);
  }
}

template <int T, int N>
__device__ inline void store(void* p, int64_t at, const float (&x)[N]) {
  typedef typename Element<T>::type E;
  constexpr int B = N * sizeof(E) < 16 ? N : 16 / sizeof(E);
  struct alignas(B * sizeof(E)) Block { E e[B]; };
#pragma unroll
  for (int i = 0; i < N; i += B) {
    Block b;
#pragma unroll
    for (int j = 0; j < B; ++j)
      b.e[j] = T == kFp32 ? (E)__float_as_uint(x[i + j]) : T == kBf16 ? (E)f2bf(x[i + j]) : (E)f2h_(x[i + j]);
    *(Block*)((E*)p + at + i) = b;
  }
}

template <int N>
__device__ inline void store_as(int type, void* p, int64_t at, const float (&x)[N]) {
  if (type == kFp16) store<kFp16, N>(p, at, x);
  else if (type == kBf16) store<kBf16, N>(p, at, x);
  else store<kFp32, N>(p, at, x);
}

}  // namespace

// Threads: tokens x parts x items of a head, items fastest: an item is V pairs, or 2 V channels that
// do not turn; a thread has its item of every parts-th head.
template <int T, int V, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int items = a.hd / (2 * V), turning = a.rd / (2 * V);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int item = (int)(id % items);
  const int part = (int)(id / items % a.parts);
  const int64_t token = id / items / a.parts;
  if (token >= a.tokens) return;
  const bool turns = item < turning;
  // where its values lie: two runs of V, or one of 2 V
  const int lo = HALF && turns ? item * V : item * 2 * V;
  const int hi = HALF && turns ? lo + a.rd / 2 : lo + V;
  float c[V], s[V];
  if (turns) {
    const int64_t pos = a.positions64 ? ((const int64_t*)a.positions)[token]
                                      : (int64_t)((const int32_t*)a.positions)[token];
    const uint64_t by = a.inverse ? (uint64_t)0 - (uint64_t)pos : (uint64_t)pos;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      cos_sin(by * a.turns[item * V + i], c[i], s[i]);
      c[i] *= a.amplitude;
      s[i] *= a.amplitude;
    }
  }
  const int heads = a.heads[0] + a.heads[1];
  for (int head = part; head < heads; head += a.parts) {
    const bool key = head >= a.heads[0];
    const int h = key ? head - a.heads[0] : head;
    const void* in = key ? a.in[1] : a.in[0];
    void* out = key ? a.out[1] : a.out[0];
    const int64_t from = token * (key ? a.in_stride[1] : a.in_stride[0]) + (int64_t)h * a.hd;
    const int64_t to = token * (key ? a.out_stride[1] : a.out_stride[0]) + (int64_t)h * a.hd;
    const int type = key ? a.out_type[1] : a.out_type[0];
    float x[V], y[V];
    load<T, V>(in, from + lo, x);
    load<T, V>(in, from + hi, y);
    if (turns) {
      float u[2 * V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float p = HALF ? x[i] : 2 * i < V ? x[2 * i % V] : y[2 * i % V];
        const float q = HALF ? y[i] : 2 * i + 1 < V ? x[(2 * i + 1) % V] : y[(2 * i + 1) % V];
        u[HALF ? i : 2 * i] = __builtin_fmaf(p, c[i], -(q * s[i]));
        u[HALF ? V + i : 2 * i + 1] = __builtin_fmaf(q, c[i], p * s[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = u[i];
        y[i] = u[V + i];
      }
    }
    store_as<V>(type, out, to + lo, x);
    store_as<V>(type, out, to + hi, y);
  }
}

}  // namespace jacq

namespace {

using jacq::RotaryArgs;

thread_local std::string g_error;

int fail(int code, const std::string& msg) {
  g_error = msg;
  return code;
}

template <class F>
int guarded(F f) {  // no C++ exception leaves a C entry
  try {
    return f();
  } catch (...) {
    return JACQ_KIVI_ENOMEM;
  }
}

int size_of(int type) { return type == JACQ_ROTARY_FP32 ? 4 : 2; }
bool is_type(int type) { return type >= JACQ_ROTARY_FP16 && type <= JACQ_ROTARY_FP32; }

template <int T, int V>
void launch(const RotaryArgs& a, int layout, unsigned blocks, hipStream_t s) {
  if (layout == JACQ_ROTARY_HALF)
    hipLaunchKernelGGL((jacq::rotary_kernel<T, V, true>), dim3(blocks), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((jacq::rotary_kernel<T, V, false>), dim3(blocks), dim3(256), 0, s, a);
}

template <int T>
void launch_v(const RotaryArgs& a, int layout, int v, unsigned blocks, hipStream_t s) {
  if (v == 8) launch<T, 8>(a, layout, blocks, s);
  else if (v == 4) launch<T, 4>(a, layout, blocks, s);
  else launch<T, 1>(a, layout, blocks, s);
}

}  // namespace

extern "C" {

const char* jacq_rotary_last_error(void) { return g_error.c_str(); }

int jacq_rotary(const jacq_rotary_args* x, hipStream_t stream) {
  return guarded([&]() -> int {
    if (!x) return fail(JACQ_KIVI_EINVAL, "argument record is null");
    if (x->tokens < 0 || x->num_heads < 0 || x->num_kv_heads < 0 || x->num_heads > 65536 ||
        x->num_kv_heads > 65536)
      return fail(JACQ_KIVI_EINVAL, "tokens and heads must not be negative, heads at most 65536");
    if (x->head_dim < 2 || x->head_dim > 1024 || x->head_dim % 2)
      return fail(JACQ_KIVI_EINVAL, "head_dim must be even and in [2, 1024], got " +
                                        std::to_string(x->head_dim));
    if (x->rotary_dim < 2 || x->rotary_dim > JACQ_ROTARY_MAX_DIM || x->rotary_dim % 2 ||
        x->rotary_dim > x->head_dim)
      return fail(JACQ_KIVI_EINVAL, "rotary_dim must be even, in [2, 256] and at most head_dim, got " +
                                        std::to_string(x->rotary_dim));
    if (x->layout != JACQ_ROTARY_HALF && x->layout != JACQ_ROTARY_INTERLEAVED)
      return fail(JACQ_KIVI_EINVAL, "layout must be JACQ_ROTARY_HALF or JACQ_ROTARY_INTERLEAVED");
    if (!is_type(x->dtype) || !is_type(x->q_out_dtype) || !is_type(x->k_out_dtype))
      return fail(JACQ_KIVI_EINVAL, "values are fp16, bf16 or fp32");
    if (!std::isfinite(x->amplitude)) return fail(JACQ_KIVI_EINVAL, "amplitude must be finite");
    const int64_t rows[4] = {x->num_heads, x->num_kv_heads, x->num_heads, x->num_kv_heads};
    const int64_t strides[4] = {x->q_stride, x->k_stride, x->q_out_stride, x->k_out_stride};
    const void* ptrs[4] = {x->Q, x->K, x->Q_OUT, x->K_OUT};
    const int types[4] = {x->dtype, x->dtype, x->q_out_dtype, x->k_out_dtype};
    for (int i = 0; i < 4; ++i)
      if (rows[i] && strides[i] < rows[i] * x->head_dim)
        return fail(JACQ_KIVI_EINVAL, "a token's row must come after the one before: a stride of at "
                                      "least " + std::to_string(rows[i] * x->head_dim) + ", got " +
                                          std::to_string(strides[i]));
    if (x->tokens == 0 || x->num_heads + x->num_kv_heads == 0) return JACQ_KIVI_OK;
    if (!x->POSITIONS || !x->TURNS) return fail(JACQ_KIVI_EINVAL, "a pointer is null");
    if ((uintptr_t)x->POSITIONS % (x->positions64 ? 8 : 4))
      return fail(JACQ_KIVI_EINVAL, "positions must be aligned to their size");
    // pairs of a thread: as many as the runs' lengths and every row's alignment allow
    int v = 8;
    for (int i = 0; i < 4; ++i) {
      if (!rows[i]) continue;
      if (!ptrs[i]) return fail(JACQ_KIVI_EINVAL, "a pointer is null");
      const int size = size_of(types[i]);
      if ((uintptr_t)ptrs[i] % size)
        return fail(JACQ_KIVI_EINVAL, "pointers must be aligned to their type");
      auto fits = [&](int n) {  // runs of n values at 16 bytes, or all of them
        const int bytes = n * size < 16 ? n * size : 16;
        return (uintptr_t)ptrs[i] % bytes == 0 && strides[i] * size % bytes == 0;
      };
      while (v > 1 && !fits(v)) v = v == 8 ? 4 : 1;
    }
    while (v > 1 && (x->head_dim % (2 * v) || x->rotary_dim % (2 * v))) v = v == 8 ? 4 : 1;
    RotaryArgs a = {};
    a.in[0] = x->Q;
    a.in[1] = x->K;
    a.out[0] = x->Q_OUT;
    a.out[1] = x->K_OUT;
    for (int i = 0; i < 2; ++i) {
      a.in_stride[i] = strides[i];
      a.out_stride[i] = strides[2 + i];
      a.heads[i] = (int)rows[i];
      a.out_type[i] = types[2 + i];
    }
    a.positions = x->POSITIONS;
    a.tokens = x->tokens;
    a.hd = x->head_dim;
    a.rd = x->rotary_dim;
    a.positions64 = x->positions64 != 0;
    a.inverse = x->inverse != 0;
    a.amplitude = x->amplitude;
    for (int i = 0; i < x->rotary_dim / 2; ++i) a.turns[i] = x->TURNS[i];
    const int64_t items = x->head_dim / (2 * v), heads = (int64_t)x->num_heads + x->num_kv_heads;
    // A thread's angles are for one head where there are few threads, else for two: 48 heads of 128 in
    // fp16, us with 1, 2, 4 and 8 a thread: 64 tokens 4.0, 4.5, 5.5 and 7.7; 1024 7.8, 7.2, 7.8 and 9.4;
    // 16384 85, 75, 78 and 82.
    const int64_t all = items * heads * x->tokens;
    const int64_t each = all <= (1 << 18) ? 1 : 2;
    a.parts = (int)((heads + each - 1) / each);
    const int64_t blocks = (items * a.parts * x->tokens + 255) / 256;
    if (blocks >= 1 << 24) return fail(JACQ_KIVI_EINVAL, "too many values in one call");
    if (x->dtype == JACQ_ROTARY_FP16) launch_v<jacq::kFp16>(a, x->layout, v, (unsigned)blocks, stream);
    else if (x->dtype == JACQ_ROTARY_BF16)
      launch_v<jacq::kBf16>(a, x->layout, v, (unsigned)blocks, stream);
    else launch_v<jacq::kFp32>(a, x->layout, v, (unsigned)blocks, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return fail(JACQ_KIVI_EHIP, std::string("rotary launch failed: ") + hipGetErrorString(e));
    return JACQ_KIVI_OK;
  });
}

}  // extern "C"
