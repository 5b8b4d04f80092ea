// q8_api.hip -- host side of the 8-bit paged cache: the C ABI of include/jacq_q8.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <climits>
#include <initializer_list>
#include <string>

#include "q8_common.h"

namespace {

using jacq::q8::AppendArgs;
using jacq::q8::AttendArgs;
using jacq::q8::Geo;
using jacq::q8::Pool;

thread_local std::string g_error;

int fail(int code, const std::string& msg) {
  g_error = msg;
  return code;
}

// No C++ exception leaves a C entry.
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (...) {
    return JACQ_KIVI_ENOMEM;
  }
}

int launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return JACQ_KIVI_OK;
  return fail(JACQ_KIVI_EHIP, std::string(what) + " launch failed: " + hipGetErrorString(e));
}

int check_geometry(const jacq_q8_geometry* x) {
  if (!x) return fail(JACQ_KIVI_EINVAL, "geometry pointer is null");
  if (x->num_heads < 1 || x->num_kv_heads < 1 || x->num_heads % x->num_kv_heads != 0)
    return fail(JACQ_KIVI_EINVAL, "num_heads must be a positive multiple of num_kv_heads, got " +
                                      std::to_string(x->num_heads) + "/" +
                                      std::to_string(x->num_kv_heads));
  if (x->num_heads / x->num_kv_heads > 16)
    return fail(JACQ_KIVI_EINVAL, "query heads per kv head must be <= 16");
  if (x->num_heads > 65536) return fail(JACQ_KIVI_EINVAL, "num_heads must be <= 65536");
  if (x->head_dim != 64 && x->head_dim != 128)
    return fail(JACQ_KIVI_EINVAL, "head_dim must be 64 or 128, got " + std::to_string(x->head_dim));
  if (x->page_size != 16 && x->page_size != 32 && x->page_size != 64)
    return fail(JACQ_KIVI_EINVAL,
                "page_size must be 16, 32 or 64, got " + std::to_string(x->page_size));
  if (x->max_pages_per_seq < 1 || x->max_pages_per_seq > JACQ_Q8_MAX_PAGES_PER_SEQ)
    return fail(JACQ_KIVI_EINVAL, "max_pages_per_seq must be in [1, 16384], got " +
                                      std::to_string(x->max_pages_per_seq));
  if (x->num_pages < 1)
    return fail(JACQ_KIVI_EINVAL, "num_pages (page storage capacity) must be positive");
  if (x->codes != JACQ_Q8_INT8 && x->codes != JACQ_Q8_E4M3)
    return fail(JACQ_KIVI_EINVAL, "codes must be JACQ_Q8_INT8 or JACQ_Q8_E4M3");
  return JACQ_KIVI_OK;
}

Geo make_geo(const jacq_q8_geometry& x) {
  Geo g;
  g.nh = x.num_heads;
  g.nkv = x.num_kv_heads;
  g.hd = x.head_dim;
  g.page = x.page_size;
  g.page_log2 = x.page_size == 16 ? 4 : x.page_size == 32 ? 5 : 6;
  g.max_pages = x.max_pages_per_seq;
  g.num_pages = x.num_pages;
  g.gqa = x.num_heads / x.num_kv_heads;
  g.codes = x.codes;
  return g;
}

bool aligned(std::initializer_list<const void*> ps, uintptr_t to) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= (uintptr_t)p;
  return (bits & (to - 1)) == 0;
}

int check_pool(const jacq_q8_pool* p) {
  if (!p || !p->k_code || !p->k_scale || !p->v_code || !p->v_scale || !p->k_tail || !p->v_tail)
    return fail(JACQ_KIVI_EINVAL, "a pool pointer is null");
  if (!aligned({p->k_code, p->v_code, p->k_tail, p->v_tail}, 16) ||
      !aligned({p->k_scale, p->v_scale}, 4))
    return fail(JACQ_KIVI_EINVAL,
                "code and tail pointers must be 16-byte aligned, scale pointers 4-byte");
  return JACQ_KIVI_OK;
}

int check_batch(int32_t batch) {
  if (batch < 0 || batch > 65535)
    return fail(JACQ_KIVI_EINVAL, "batch must be in [0, 65535], got " + std::to_string(batch));
  return JACQ_KIVI_OK;
}

int check_stride(int64_t stride, int64_t row, const char* name) {
  if (stride < row || stride % 8 != 0)
    return fail(JACQ_KIVI_EINVAL, std::string(name) + " row stride must be a multiple of 8 and at "
                                      "least " + std::to_string(row) + ", got " +
                                      std::to_string(stride));
  return JACQ_KIVI_OK;
}

Pool read_pool(const jacq_q8_pool& p) {
  return {p.k_code, p.k_scale, p.v_code, p.v_scale, (const uint16_t*)p.k_tail,
          (const uint16_t*)p.v_tail};
}

// Compute units of the current device, looked up once per device.
int device_cus() {
  constexpr int kMost = 64;
  static std::atomic<int> known[kMost];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (dev >= 0 && dev < kMost)
    if (const int c = known[dev].load(std::memory_order_relaxed)) return c;
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus < 1)
    return 256;
  if (dev >= 0 && dev < kMost) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// ---- how an attention call runs ----
// The decode kernel reads the cache once per 32 rows of a kv head (a second time mostly from a
// cache nearer by) and splits it freely; the prefill kernel shares it among 128 rows.  The first is
// used up to 64 rows, and for so few rows in all that the second leaves most of the chip idle.
// Decode against prefill, us (heads of 128 unless said otherwise):
//   40 to 64 rows  32 sequences, 64/8 heads, 8 queries: of 500 tokens 26 against 29, 2000 48
//                  against 58, 12000 222 against 279; 4 of 16384, 40/8 heads, 12 queries: 61
//                  against 59; 64 of 500, 32/8 heads, 16 queries: 45 against 37
//   70, 80 rows    4 of 16384, 40/8 heads, 16 queries: 76 against 64; 16 of 4096, 14/2 heads of 64,
//                  14 queries: 34 against 27
//   one sequence   40/8 heads, 32 queries: of 2048 tokens 20 against 27, 16384 45 against 49; 8/1
//                  heads, 16384 tokens: 128 queries 34 against 41, 200 53 against 49
constexpr int kFewRows = 64;
constexpr int kFewHeads = 2048;  // queries x query heads of the call
// Units up to which the decode kernel does not cut a segment: no plan, no join.  The table's width
// bounds them.  40/8 heads of 128, without against with (us): one sequence of 700 tokens 14.5
// against 15.8, 16 of 500 14.6 against 18.1, 64 of 500 22.9 against 27.0.
constexpr int kWholeUnits = 16;
// Sequences up to which every workgroup finds the cut by itself (a lane each); more have a kernel
// for it.  32/8 heads of 128, by itself against by the kernel (us): 80 sequences of 100 to 4000
// tokens 99 against 97, 256 of 100 to 1000 99 against 86, 512 of 100 to 500 187 against 123.
constexpr int kCutBatch = 64;

struct Plan {
  bool prefill, planned;
  float load;
  int slices, nb, rows, row_blocks, target, groups;
  size_t ml, acc, plan, group_lse, row_lse, bytes;  // offsets into the workspace, and its size
};

// A prefill's slices, for as many tokens as the table addresses: the kernels use fewer for
// sequences of fewer (slices_cost, which has the reasons).  One, unless more promise 3 % at least:
// where a CU has many row tiles the promise is no more than a fuller last round, and the slices that
// are not used and the merge cost more (64 prompts of 100 to 500 tokens under a table of 65536, 32/8
// heads of 128, 18.8 tiles a CU: 227 us in up to 4 slices, 190 in one).
int plan_slices(float load, int64_t tokens) {
  const int most =
      (int)std::min<int64_t>(jacq::kMaxSlices, tokens / (jacq::kSliceUnits * jacq::kTile));
  auto cost = [&](int s) { return jacq::slices_cost(load, s, (float)tokens); };
  int best = 1;
  for (int s = 2; s <= most; ++s)
    if (cost(s) < cost(best)) best = s;
  return cost(best) < 0.97f * cost(1) ? best : 1;
}

Plan plan_attend(const Geo& g, int batch, int total_q, int max_q, bool weighted) {
  Plan p = {};
  const int64_t rows = (int64_t)max_q * g.gqa;
  // The call's queries, not max_q for every sequence: of a cache's sequences some may have none.
  const int64_t queries = std::min<int64_t>((int64_t)batch * max_q, total_q);
  // Their row tiles, or blocks of so many rows: of as few sequences as they can be of, and a begun
  // one more for each but the first, as most calls of several are ragged.
  auto blocks = [&](int64_t block) {
    const int64_t each = (rows + block - 1) / block, full = queries / max_q, rest = queries % max_q;
    return std::min(batch * each, full * each + (rest * g.gqa + block - 1) / block +
                                      full + (rest > 0) - 1);
  };
  p.prefill = !weighted && rows > kFewRows && queries * g.nh > kFewHeads;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (p.prefill) {
    p.load = (float)(blocks(jacq::kPrefillRows) * g.nkv) / (float)device_cus();
    p.slices = plan_slices(p.load, (int64_t)g.max_pages * g.page);
    if (p.slices > 1) {
      const size_t rows_all = (size_t)p.slices * total_q * g.nh;
      p.ml = take(rows_all * 2 * sizeof(float));
      p.acc = take(rows_all * g.hd * sizeof(float));
    }
    p.bytes = at;
    return p;
  }
  p.nb = rows <= 16 ? 1 : 2;
  p.rows = (int)std::min<int64_t>(rows, 16 * p.nb);
  p.row_blocks = (int)((rows + 16 * p.nb - 1) / (16 * p.nb));
  p.groups = g.max_pages * (g.page / 16);
  const int64_t most = ((int64_t)p.groups + 3) / 4 + 1;  // units of a segment at most
  const int64_t segments = (int64_t)batch * g.nkv * p.row_blocks;
  if (most > kWholeUnits) {
    const int64_t slots = (int64_t)jacq::q8::decode_groups(g.hd, p.nb) * device_cus();
    // one round of workgroups where the segments' last slices are at most a sixth of it, else two:
    // with one, 16 sequences of 1000 to 8000, 32/32 heads of 128, take 116 us instead of 111
    p.target = (int)(3 * blocks(16 * p.nb) * g.nkv <= slots ? slots : 2 * slots);
  }
  const size_t parts = p.target ? (size_t)p.target + segments : 0;
  p.ml = take(parts * p.rows * 2 * sizeof(float));
  p.acc = take(parts * p.rows * g.hd * sizeof(float));
  p.planned = p.target && batch > kCutBatch;
  p.plan = take(p.planned ? ((size_t)batch + 2) * sizeof(int32_t) : 0);
  p.group_lse = take(weighted ? (size_t)segments * p.groups * p.rows * sizeof(float) : 0);
  p.row_lse = take(weighted ? (size_t)total_q * g.nh * sizeof(float) : 0);
  p.bytes = at;
  return p;
}

// As many units as Place may give to the call's queries.
int64_t place_units(const AttendArgs& a, int per, int log2) {
  const int64_t of_all = ((int64_t)a.total_q * per >> log2) + a.batch;
  const int64_t each = ((int64_t)a.max_q * per + (1 << log2) - 1) >> log2;
  return a.batch <= jacq::kCounted ? std::min(of_all, a.batch * each) : of_all;
}

}  // namespace

extern "C" {

int jacq_q8_version(void) { return JACQ_Q8_VERSION; }

const char* jacq_q8_last_error(void) { return g_error.c_str(); }

int jacq_q8_check_geometry(const jacq_q8_geometry* geo) {
  return guarded([&] { return check_geometry(geo); });
}

int64_t jacq_q8_max_seq_len(const jacq_q8_geometry* geo) {
  return geo ? (int64_t)geo->max_pages_per_seq * geo->page_size : 0;
}

int jacq_q8_append(const jacq_q8_geometry* geo, const jacq_q8_pool* pool, const void* NEW_K,
                   const void* NEW_V, int32_t dtype, int64_t k_stride, int64_t v_stride,
                   const int32_t* CU_NEW, const int32_t* START_LENS,
                   const int32_t* BLOCK_TABLES, int32_t total_new, int32_t max_new,
                   int32_t batch, hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_pool(pool)) return e;
    if (int e = check_batch(batch)) return e;
    if (dtype != JACQ_Q8_FP16 && dtype != JACQ_Q8_BF16)
      return fail(JACQ_KIVI_EINVAL, "new tokens must be fp16 or bf16");
    if (total_new < 0 || max_new < 0) return fail(JACQ_KIVI_EINVAL, "negative number of tokens");
    if (!CU_NEW && (total_new != batch || (batch && max_new != 1)))
      return fail(JACQ_KIVI_EINVAL, "without CU_NEW every sequence has one new token");
    const int64_t row = (int64_t)geo->num_kv_heads * geo->head_dim;
    if (int e = check_stride(k_stride, row, "NEW_K")) return e;
    if (int e = check_stride(v_stride, row, "NEW_V")) return e;
    if (batch == 0 || total_new == 0 || max_new == 0) return JACQ_KIVI_OK;
    if (!NEW_K || !NEW_V || !START_LENS || !BLOCK_TABLES)
      return fail(JACQ_KIVI_EINVAL, "a tensor pointer is null");
    if (!aligned({NEW_K, NEW_V}, 16) || !aligned({CU_NEW, START_LENS, BLOCK_TABLES}, 4))
      return fail(JACQ_KIVI_EINVAL, "token pointers must be 16-byte aligned, tables 4-byte");
    AppendArgs a = {*pool,      (const uint16_t*)NEW_K, (const uint16_t*)NEW_V, k_stride, v_stride,
                    CU_NEW,     START_LENS,             BLOCK_TABLES,           total_new,
                    std::min(max_new, total_new),       dtype == JACQ_Q8_BF16};
    // more tokens than the table addresses are dropped anyway
    a.max_new = std::min(a.max_new, geo->max_pages_per_seq * geo->page_size);
    if ((int64_t)geo->num_kv_heads * (a.max_new / geo->page_size + 1) > INT32_MAX)
      return fail(JACQ_KIVI_EINVAL, "too many blocks in one append");
    return launched(jacq::q8::launch_append(make_geo(*geo), a, batch, stream), "append");
  });
}

size_t jacq_q8_attend_workspace_size(const jacq_q8_geometry* geo, int32_t batch, int32_t total_q,
                                     int32_t max_q, int32_t weighted) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (batch > 0 && total_q > 0 && max_q > 0)
      bytes = plan_attend(make_geo(*geo), batch, total_q, std::min(max_q, total_q), weighted != 0)
                  .bytes;
    return JACQ_KIVI_OK;
  });
  return bytes;
}

int jacq_q8_attend(const jacq_q8_geometry* geo, const jacq_q8_pool* pool,
                   const jacq_q8_attend_args* x, void* workspace, size_t workspace_bytes,
                   hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_pool(pool)) return e;
    if (!x) return fail(JACQ_KIVI_EINVAL, "argument record is null");
    if (int e = check_batch(x->batch)) return e;
    if (x->q_dtype != JACQ_Q8_FP16 && x->q_dtype != JACQ_Q8_BF16)
      return fail(JACQ_KIVI_EINVAL, "queries must be fp16 or bf16");
    if (x->o_dtype != x->q_dtype && x->o_dtype != JACQ_Q8_FP32)
      return fail(JACQ_KIVI_EINVAL, "the output is of the queries' type or fp32");
    if (x->total_q < 0 || x->max_q < 0) return fail(JACQ_KIVI_EINVAL, "negative number of queries");
    if (!x->CU_Q && (x->total_q != x->batch || (x->batch && x->max_q != 1)))
      return fail(JACQ_KIVI_EINVAL, "without CU_Q every sequence has one query");
    if (x->window < 0 || x->sinks < 0)
      return fail(JACQ_KIVI_EINVAL, "window and sinks must not be negative");
    if (!std::isfinite(x->scale) || x->scale <= 0 || !std::isfinite(x->decay) || x->decay < 0)
      return fail(JACQ_KIVI_EINVAL, "scale must be positive and finite, decay not negative");
    if (x->WEIGHTS && x->max_q > JACQ_Q8_MAX_WEIGHTED_QUERIES)
      return fail(JACQ_KIVI_EINVAL, "block weights take at most 64 queries per sequence, got " +
                                        std::to_string(x->max_q));
    const int64_t row = (int64_t)geo->num_heads * geo->head_dim;
    if (int e = check_stride(x->q_stride, row, "Q")) return e;
    if (x->batch == 0) return JACQ_KIVI_OK;
    const bool none = x->total_q == 0 || x->max_q == 0;  // then there are offsets, not one query each
    if (none && !x->WEIGHTS) return JACQ_KIVI_OK;
    if (!x->SEQ_LENS || (!none && (!x->Q || !x->O || !x->BLOCK_TABLES)))
      return fail(JACQ_KIVI_EINVAL, "a tensor pointer is null");
    if (!aligned({x->Q, x->O, workspace}, 16) ||
        !aligned({x->CU_Q, x->SEQ_LENS, x->BLOCK_TABLES, x->LSE, x->WEIGHTS}, 4))
      return fail(JACQ_KIVI_EINVAL,
                  "Q, O and workspace pointers must be 16-byte aligned, the others 4-byte");
    const Geo g = make_geo(*geo);
    AttendArgs a = {};
    a.pool = read_pool(*pool);
    a.q = (const uint16_t*)x->Q;
    a.cu = x->CU_Q;
    a.lens = x->SEQ_LENS;
    a.tables = x->BLOCK_TABLES;
    a.o = x->O;
    a.lse = x->LSE;
    a.weights = x->WEIGHTS;
    a.q_stride = x->q_stride;
    a.q_bf16 = x->q_dtype == JACQ_Q8_BF16;
    a.o_type = x->o_dtype;
    a.batch = x->batch;
    a.total_q = x->total_q;
    a.max_q = std::min(x->max_q, x->total_q);
    a.window = std::min(x->window, 1 << 30);
    a.sinks = std::min(x->sinks, 1 << 30);
    a.scale = x->scale * jacq::kLog2e;
    a.decay = x->decay;
    if (none) {
      a.groups = g.max_pages * (g.page / 16);
      return launched(jacq::q8::launch_decay(g, a, stream), "decay");
    }
    const Plan p = plan_attend(g, a.batch, a.total_q, a.max_q, a.weights != nullptr);
    if ((int64_t)a.max_q * g.gqa > INT32_MAX / 2 ||
        (int64_t)a.batch * g.nkv * std::max(1, p.row_blocks) > INT32_MAX)
      return fail(JACQ_KIVI_EINVAL, "too many query rows in one call");
    if (p.bytes && (!workspace || workspace_bytes < p.bytes))
      return fail(JACQ_KIVI_ENOMEM, "the workspace needs " + std::to_string(p.bytes) +
                                        " bytes, got " +
                                        std::to_string(workspace ? workspace_bytes : 0));
    uint8_t* ws = (uint8_t*)workspace;
    a.part_ml = (float*)(ws + p.ml);
    a.part_acc = (float*)(ws + p.acc);
    a.group_lse = a.weights ? (float*)(ws + p.group_lse) : nullptr;
    a.row_lse = a.weights ? (float*)(ws + p.row_lse) : nullptr;
    a.slices = p.slices;
    a.load = p.load;
    const int64_t tiles = place_units(a, g.gqa, jacq::kRowsLog2);
    const int64_t merges = p.slices > 1 ? place_units(a, g.nh, jacq::merge_log2(g.hd)) : 0;
    // a launch has fewer than 2^32 threads
    if (p.prefill && std::max(tiles * g.nkv, merges) >= 1 << 24)
      return fail(JACQ_KIVI_EINVAL, "too many query rows in one call");
    a.tiles = (unsigned)tiles;
    a.merges = (unsigned)merges;
    if (p.prefill) return launched(jacq::q8::launch_prefill(g, a, stream), "prefill");
    a.target = p.target;
    a.cus = device_cus();
    a.plan = p.planned ? (int32_t*)(ws + p.plan) : nullptr;
    a.rows = p.rows;
    a.row_blocks = p.row_blocks;
    a.groups = p.groups;
    return launched(jacq::q8::launch_decode(g, a, p.nb, stream), "decode");
  });
}

int jacq_q8_read(const jacq_q8_geometry* geo, const jacq_q8_pool* pool, const int32_t* STARTS,
                 const int32_t* ENDS, const int32_t* BLOCK_TABLES, int32_t batch, int32_t total,
                 void* K, void* V, int32_t dtype, hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_pool(pool)) return e;
    if (int e = check_batch(batch)) return e;
    if (dtype < JACQ_Q8_FP16 || dtype > JACQ_Q8_FP32)
      return fail(JACQ_KIVI_EINVAL, "values are read as fp16, bf16 or fp32");
    if (total < 0) return fail(JACQ_KIVI_EINVAL, "negative number of tokens");
    if (batch == 0 || total == 0) return JACQ_KIVI_OK;
    if (!STARTS || !ENDS || !BLOCK_TABLES || !K || !V)
      return fail(JACQ_KIVI_EINVAL, "a tensor pointer is null");
    if (!aligned({K, V}, 16) || !aligned({STARTS, ENDS, BLOCK_TABLES}, 4))
      return fail(JACQ_KIVI_EINVAL, "K and V must be 16-byte aligned, tables 4-byte");
    if ((int64_t)geo->num_kv_heads * (total / 16 + 2 * batch) > INT32_MAX)
      return fail(JACQ_KIVI_EINVAL, "too many tokens in one read");
    return launched(jacq::q8::launch_read(make_geo(*geo), read_pool(*pool), STARTS, ENDS,
                                          BLOCK_TABLES, batch, total, K, V, dtype, stream),
                    "read");
  });
}

int jacq_q8_evict(const jacq_q8_geometry* geo, const float* WEIGHTS, const int32_t* SEQ_LENS,
                  const int32_t* BLOCK_TABLES, int32_t batch, int32_t keep, int32_t sink_pages,
                  int32_t recent_pages, int32_t* TABLES_OUT, int32_t* LENS_OUT,
                  float* WEIGHTS_OUT, int32_t* EVICTED, hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_batch(batch)) return e;
    if (sink_pages < 0 || recent_pages < 0 || keep < 0 ||
        (int64_t)sink_pages + recent_pages > keep)
      return fail(JACQ_KIVI_EINVAL,
                  "keep must be at least sink_pages + recent_pages, neither negative; got " +
                      std::to_string(keep) + ", " + std::to_string(sink_pages) + ", " +
                      std::to_string(recent_pages));
    if (batch == 0) return JACQ_KIVI_OK;
    if (!WEIGHTS || !SEQ_LENS || !BLOCK_TABLES || !TABLES_OUT || !LENS_OUT || !WEIGHTS_OUT ||
        !EVICTED)
      return fail(JACQ_KIVI_EINVAL, "a tensor pointer is null");
    if (!aligned({WEIGHTS, SEQ_LENS, BLOCK_TABLES, TABLES_OUT, LENS_OUT, WEIGHTS_OUT, EVICTED}, 4))
      return fail(JACQ_KIVI_EINVAL, "tensor pointers must be 4-byte aligned");
    return launched(
        jacq::q8::launch_evict(make_geo(*geo), WEIGHTS, SEQ_LENS, BLOCK_TABLES, batch, keep,
                               sink_pages, recent_pages, TABLES_OUT, LENS_OUT, WEIGHTS_OUT, EVICTED,
                               stream),
        "evict");
  });
}

}  // extern "C"
