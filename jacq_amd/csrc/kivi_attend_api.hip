// kivi_attend_api.hip -- host side of the int4 cache's attention of chunks and of its read-back: the
// C ABI of include/jacq_kivi_attend.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "jacq_kivi_attend.h"
#include "kivi_attend.h"
#include "kivi_kernels.h"

namespace {

using jacq::KiviAttendArgs;
using jacq::KiviGeo;
using jacq::KiviPool;

static_assert(jacq::kFp16 == JACQ_KIVI_FP16 && jacq::kBf16 == JACQ_KIVI_BF16 &&
                  jacq::kFp32 == JACQ_KIVI_FP32,
              "types");

int fail(const std::string& msg) { return jacq::set_last_error(JACQ_KIVI_EINVAL, msg); }

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
  return jacq::set_last_error(JACQ_KIVI_EHIP,
                              std::string(what) + " launch failed: " + hipGetErrorString(e));
}

bool aligned(std::initializer_list<const void*> ps, uintptr_t to) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= (uintptr_t)p;
  return (bits & (to - 1)) == 0;
}

KiviGeo make_geo(const jacq_kivi_geometry& x) {
  KiviGeo g;
  g.nh = x.num_heads;
  g.nkv = x.num_kv_heads;
  g.hd = x.head_dim;
  g.page = x.page_size;
  g.residual = x.residual;
  g.max_pages = x.max_pages_per_seq;
  g.num_pages = x.num_pages;
  g.gqa = x.num_heads / x.num_kv_heads;
  g.rs = x.residual + jacq::kGroup;
  g.lq = (int)(((int64_t)x.max_pages_per_seq * x.page_size / jacq::kGroup) * jacq::kGroup);
  return g;
}

int check_geometry(const jacq_kivi_geometry* x) {
  if (int e = jacq_kivi_check_geometry(x)) return e;
  if (x->num_heads > 65536) return fail("num_heads must be <= 65536");
  return JACQ_KIVI_OK;
}

int check_pool(const jacq_kivi_pool* p) {
  if (!p || !p->k_code || !p->k_scale || !p->k_zero || !p->v_code || !p->v_scale || !p->v_zero ||
      !p->k_scratch || !p->v_scratch)
    return fail("a pool pointer is null");
  if (!aligned({p->k_code, p->k_scale, p->k_zero, p->v_code, p->v_scale, p->v_zero, p->k_scratch,
                p->v_scratch},
               16))
    return fail("pool pointers must be 16-byte aligned");
  return JACQ_KIVI_OK;
}

int check_batch(int32_t batch) {
  if (batch < 0 || batch > 65535)
    return fail("batch must be in [0, 65535], got " + std::to_string(batch));
  return JACQ_KIVI_OK;
}

KiviPool read_pool(const jacq_kivi_pool& p) {
  return {p.k_code, p.k_scale, p.k_zero, p.v_code, p.v_scale, p.v_zero, p.k_scratch, p.v_scratch};
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
// Units (of 32 tokens) up to which segments stay whole: no plan, no join, a launch less.  The table's
// width bounds them, the lengths are the device's.  us a call, whole against cut:
//   kWholeUnits     one of 512 tokens, 2 queries, 32/4 heads of 64 8.8 and 12.3; of 700 (24 units), 4 queries,
//                   40/8 heads of 128 14.6 and 14.0; of 1500 22.2 and 13.9
//   kWholeFull      where every CU has two segments: 32 of 300 to 1500, 16/16 heads of 64 20.2 and 23.4; 256,
//                   14/2 heads of 64 21.5 and 27.4; 64 of 1500 to 1900, 32/8 heads of 128 36 and 41; but one
//                   of 1500 among 63 of 30 19.5 and 14.3
constexpr int kWholeUnits = 24, kWholeFull = 64;
// Sequences up to which every workgroup finds the cut by itself (a lane each); more have a kernel
// for it, 2 us a call where both could.
constexpr int kCutBatch = 64;

// A call is a prompt's, whose tokens become fp16 once, in the workspace, from so many rows of a kv head
// and (query, head) rows x tokens of the table on.  Few-query kernel against prompts', us a call:
//   160 rows   8 sequences of 4000 to 8000, 40/8 heads of 128 121 against 138; 32 of 300 to 1500 77 and 92
//   320 rows   the same 171 and 164, 131 and 117; one of 16384 62 and 69 (42 M rows x tokens), 16/16 heads
//              of 64 83 and 69 (84 M)
//   640 rows   one of 16384, 40/8 heads of 128 107 and 92 (84 M), of 700 19 and 28 (4 M); 8 of 4000 to
//              8000, 14/2 heads of 64 91 and 57 (82 M), 32 of 300 to 1500 50 and 46 (61 M)
//   1274 rows  one of 16384, 14/2 heads of 64 45 and 48 (42 M)
// or from so many full rounds of the few-query kernel's workgroups on, each of which pays its start and end:
// prompts of 16 sequences of 200 tokens, 32/8 heads of 128 (3200 workgroups, 6 rounds), 57 and 39 us, of 8 of
// 300 (2432) 50 and 36, of 4 of 300 to 600 46 and 35; but 128 queries of each of 8 of 500 to 1000, 40/8 heads
// (1280), 49 and 55, a prompt of 1000 (1256) 43 and 49.
constexpr int64_t kPromptRows = 320;
constexpr int64_t kPromptWork = 50000000;
constexpr int64_t kPromptRounds = 3;
// Where a call has at most half the queries that max_q for every sequence would be, as with chunks of some
// prompts between steps of other sequences, those of at most so many rows of a kv head are the few-query
// kernel's, which lays nothing.  40/8 heads of 128, sequences of 4000 tokens, us with the split and without:
// 512 queries of one of 32 143 and 345, of two of 64 212 and 635, of one of 3 93 and 86; 7 of 16 365 and 398.
// 16 rows would do for single queries (136, 201, 92), not for four of them.
constexpr int kSplitRows = 32;
// Such a call is a prompt's from so many segments of the few-query kernel on, too, since most are empty:
// 256 queries of one of 64 sequences of 1000 tokens (20480) 111 us there and 63 so, of one of 32 (10240) 66
// and 58, of one of 16 (5120) 43 and 57; 100 of each of 4 of 100 of 200 tokens (10400) 36 and 43.
constexpr int64_t kSplitSegments = 12000;
// Bytes of fp16 tiles that a pass lays in the workspace, about.
constexpr int64_t kPassBytes = (int64_t)1 << 31;
// Passes up to which a call is a prompt's: the table's width tells how many there may be, and one with nothing
// to do still takes 9 to 12 us.  256 sequences, 40/8 heads of 128, us in the few-query kernel and in passes: 200
// queries of each of 1000 tokens, 33 passes, 2228 and 1847, 130 passes 2224 and 3203; of 65 passes 500 of 1000
// 5025 and 4287, 200 of 3000 5605 and 4975, but 200 of 200 1056 and 1379, 70 of 1000 958 and 1438.
constexpr int64_t kMostPasses = 64;
// Of a call that can be split there are more passes where the few-query kernel has so many segments for each:
// most of them are empty, and still cost 2 ns, and it leaves segments whole (kMostParts).  A chunk beside single
// queries of 2047 sequences, table of 131072 tokens, 40/8 heads of 128, us there and in passes, the others of
// 1000 to 4000 tokens and of 100 to 200:
//   64 queries, 2200 segments a pass    2694 and 2692, 634 and 1395
//   128, 4200                           5078 and 3093, 1216 and 1820
//   256, 8000                           5415 and 3266, 1550 and 1917
//   512, 14400                          6076 and 3452, 2239 and 2076
// of 255 sequences, 65 passes: 2048 queries, 10000 segments a pass, 1384 and 916.
constexpr int64_t kPassSegments = 4000;
// A prompt's workgroups a CU at most, slices counted: those that the lengths do not ask for end at once.
constexpr int64_t kMostGroups = 8;
// Bytes of parts for which the few-query kernel still cuts.  A call of more has 64 thousand segments (of 32 rows
// of 128), which fill the CUs though some are empty; but a long one among them stays whole.
constexpr int64_t kMostParts = (int64_t)1 << 30;

// Workgroups of a launch, which has fewer than 2^32 threads.
constexpr int64_t kMostSegments = 1 << 24;

// Test hook: not 0: the bytes of a pass on the calling thread.
thread_local int64_t g_pass_bytes = 0;

struct Plan {
  bool prompt, few;       // which kernels run: both for sequences of many queries and of few
  int split;              // then, the queries up to which a sequence is the few-query kernel's
  bool planned;
  int nb, rows, row_blocks, target;
  int slices, per_pass, passes;
  size_t ml, acc, plan, slots, images, poison, bytes;  // offsets into the workspace, and its size
  size_t few_ml, few_acc;
};

Plan plan_attend(const KiviGeo& g, int batch, int total_q, int max_q) {
  Plan p = {};
  const int64_t rows = (int64_t)max_q * g.gqa;
  // The call's queries, not max_q for every sequence: of a cache's sequences some may have none.
  const int64_t queries = std::min<int64_t>((int64_t)batch * max_q, total_q);
  // Their blocks of so many rows: of as few sequences as they can be of, and a begun one more for
  // each but the first, as most calls of several are ragged.
  auto blocks = [&](int64_t block) {
    const int64_t each = (rows + block - 1) / block, full = queries / max_q, rest = queries % max_q;
    return std::min(batch * each, full * each + (rest * g.gqa + block - 1) / block +
                                      full + (rest > 0) - 1);
  };
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t tokens = (int64_t)g.lq + g.residual;
  const int64_t cap = (tokens + jacq::kTile - 1) / jacq::kTile;  // images of a sequence and kv head
  const int64_t image = (int64_t)4 * jacq::kTile * g.hd * g.nkv;
  const int64_t pass_bytes = g_pass_bytes ? g_pass_bytes : kPassBytes;
  if (2 * (int64_t)total_q <= (int64_t)batch * max_q) p.split = kSplitRows / g.gqa;
  const int64_t images = std::min<int64_t>(batch, total_q / (p.split + 1)) * cap;
  p.per_pass = (int)std::max<int64_t>(1, std::min(images, pass_bytes / image));
  const int64_t passes = (images + p.per_pass - 1) / p.per_pass;
  const int64_t segments = (int64_t)batch * g.nkv * ((rows + 31) / 32);  // of the few-query kernel alone
  const bool pays = rows >= kPromptRows &&
                    (passes <= kMostPasses || (p.split && passes * kPassSegments <= segments)) &&
                    (queries * g.nh * tokens >= kPromptWork ||
                     blocks(32) * g.nkv >= kPromptRounds * jacq::few_groups(g.hd, 2) * device_cus() ||
                     (p.split && segments >= kSplitSegments));
  // more segments than a launch takes: row tiles are of the call's queries alone, and four times as long
  p.prompt = images > 0 && images <= INT32_MAX - 4096 && (pays || segments >= kMostSegments);
  p.few = !p.prompt || p.split;
  if (p.prompt) {
    p.passes = (int)passes;
    // row tiles in so many slices that their workgroups are no more than kMostGroups a CU: the device
    // uses as many as the lengths ask for (kivi_slots_kernel), the others end at once
    const int64_t groups = std::max<int64_t>(1, blocks(jacq::kPrefillRows) * g.nkv);
    p.slices = (int)std::max<int64_t>(
        1, std::min<int64_t>({jacq::kMaxSlices, tokens / (jacq::kSliceUnits * jacq::kTile),
                              kMostGroups * device_cus() / groups}));
    if (p.slices > 1) {
      const size_t rows_all = (size_t)p.slices * total_q * g.nh;
      p.ml = take(rows_all * 2 * sizeof(float));
      p.acc = take(rows_all * g.hd * sizeof(float));
    }
    // a sequence's images may end behind the pass that they begin in
    const size_t held = (size_t)(passes == 1 ? images : p.per_pass + cap) * g.nkv;
    p.slots = take(((size_t)batch + 2) * sizeof(int32_t));
    p.poison = take(held * sizeof(uint64_t));
    p.images = take(held * 4 * jacq::kTile * g.hd);
  }
  if (p.few) {
    const int64_t most_rows = p.prompt ? p.split * g.gqa : rows;
    p.nb = most_rows <= 16 ? 1 : 2;
    p.rows = (int)std::min<int64_t>(most_rows, 16 * p.nb);
    p.row_blocks = (int)((most_rows + 16 * p.nb - 1) / (16 * p.nb));
    const int64_t most = (g.lq + g.residual + jacq::kGroup - 1) / jacq::kGroup;  // units of a segment
    const int64_t segments = (int64_t)batch * g.nkv * p.row_blocks;
    if (most > (segments >= 2 * device_cus() ? kWholeFull : kWholeUnits)) {
      const int64_t slots = (int64_t)jacq::few_groups(g.hd, p.nb) * device_cus();
      const int64_t filled = p.prompt ? segments : blocks(16 * p.nb) * g.nkv;
      // One round of workgroups, or two where one would have fewer than two slices of a segment.  us with a
      // third as the border, and with a half: 24, 28 and 32 sequences of 1500 to 6007, 4 queries, 40/8 heads
      // of 128, 53 and 45, 54 and 49, 58 and 56 (all of 4000: 45 and 50, 54 and 54, 55 and 56); 144 of 1000
      // to 4000, 14/2 heads of 64, 40 and 37.  With one round always, 64 of the first take 104 and not 95.
      p.target = (int)(2 * filled <= slots ? slots : 2 * slots);
    }
    if (segments >= kMostSegments ||  // a call that is refused
        (p.target + segments) * p.rows * (g.hd + 2) * (int64_t)sizeof(float) > kMostParts)
      p.target = 0;
    const size_t parts = p.target ? (size_t)p.target + segments : 0;
    p.few_ml = take(parts * p.rows * 2 * sizeof(float));
    p.few_acc = take(parts * p.rows * g.hd * sizeof(float));
    p.planned = p.target && batch > kCutBatch;
    p.plan = take(p.planned ? ((size_t)batch + 2) * sizeof(int32_t) : 0);
  }
  p.bytes = at;
  return p;
}

// As many units as Place may give to the call's queries.
int64_t place_units(const KiviAttendArgs& a, int per, int log2) {
  const int64_t of_all = ((int64_t)a.total_q * per >> log2) + a.batch;
  const int64_t each = ((int64_t)a.max_q * per + (1 << log2) - 1) >> log2;
  return a.batch <= jacq::kCounted ? std::min(of_all, a.batch * each) : of_all;
}

}  // namespace

extern "C" {

// Test hooks outside the ABI: prompts of the calling thread lay about so many bytes of fp16 tiles a
// pass (0: as many as ever); whether a call is a prompt's.
void jacq_kivi_test_pass_bytes(int64_t bytes) { g_pass_bytes = bytes; }
int32_t jacq_kivi_test_is_prompt(const jacq_kivi_geometry* geo, int32_t batch, int32_t total_q,
                                 int32_t max_q) {
  return plan_attend(make_geo(*geo), batch, total_q, std::min(max_q, total_q)).prompt;
}

size_t jacq_kivi_attend_workspace_size(const jacq_kivi_geometry* geo, int32_t batch, int32_t total_q,
                                       int32_t max_q) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (batch > 0 && total_q > 0 && max_q > 0)
      bytes = plan_attend(make_geo(*geo), batch, total_q, std::min(max_q, total_q)).bytes;
    return JACQ_KIVI_OK;
  });
  return bytes;
}

int jacq_kivi_attend(const jacq_kivi_geometry* geo, const jacq_kivi_pool* pool,
                     const jacq_kivi_attend_args* x, void* workspace, size_t workspace_bytes,
                     hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_pool(pool)) return e;
    if (!x) return fail("argument record is null");
    if (int e = check_batch(x->batch)) return e;
    if (x->q_dtype != JACQ_KIVI_FP16 && x->q_dtype != JACQ_KIVI_BF16)
      return fail("queries must be fp16 or bf16");
    if (x->o_dtype != x->q_dtype && x->o_dtype != JACQ_KIVI_FP32)
      return fail("the output is of the queries' type or fp32");
    if (x->total_q < 0 || x->max_q < 0) return fail("negative number of queries");
    if (!x->CU_Q && (x->total_q != x->batch || (x->batch && x->max_q != 1)))
      return fail("without CU_Q every sequence has one query");
    if (x->window < 0 || x->sinks < 0) return fail("window and sinks must not be negative");
    if (x->causal != 0 && x->causal != 1) return fail("causal must be 0 or 1");
    if (!x->causal && (x->window || x->sinks))
      return fail("queries that see every token have no window and no sinks");
    if (!std::isfinite(x->scale * jacq::kLog2e) || x->scale <= 0)
      return fail("scale must be positive and finite, times log2(e) too");
    const int64_t row = (int64_t)geo->num_heads * geo->head_dim;
    if (x->q_stride < row || x->q_stride % 8 != 0)
      return fail("Q row stride must be a multiple of 8 and at least " + std::to_string(row) +
                  ", got " + std::to_string(x->q_stride));
    if (x->batch == 0 || x->total_q == 0 || x->max_q == 0) return JACQ_KIVI_OK;
    if (!x->Q || !x->O || !x->SEQ_LENS || (!x->BLOCK_TABLES && geo->max_pages_per_seq > 0))
      return fail("a tensor pointer is null");
    if (!aligned({x->Q, x->O, workspace}, 16) ||
        !aligned({x->CU_Q, x->SEQ_LENS, x->BLOCK_TABLES, x->LSE}, 4))
      return fail("Q, O and workspace pointers must be 16-byte aligned, the others 4-byte");
    const KiviGeo g = make_geo(*geo);
    KiviAttendArgs a = {};
    a.pool = read_pool(*pool);
    a.q = (const uint16_t*)x->Q;
    a.cu = x->CU_Q;
    a.lens = x->SEQ_LENS;
    a.tables = x->BLOCK_TABLES;
    a.o = x->O;
    a.lse = x->LSE;
    a.q_stride = x->q_stride;
    a.q_bf16 = x->q_dtype == JACQ_KIVI_BF16;
    a.o_type = x->o_dtype;
    a.batch = x->batch;
    a.total_q = x->total_q;
    a.max_q = std::min(x->max_q, x->total_q);
    a.window = std::min(x->window, 1 << 30);
    a.sinks = std::min(x->sinks, 1 << 30);
    a.causal = x->causal;
    a.scale = x->scale * jacq::kLog2e;
    const Plan p = plan_attend(g, a.batch, a.total_q, a.max_q);
    const int64_t segments = (int64_t)a.batch * g.nkv * p.row_blocks;
    const int64_t tiles = place_units(a, g.gqa, jacq::kRowsLog2);
    const int64_t merges = p.slices > 1 ? place_units(a, g.nh, jacq::merge_log2(g.hd)) : 0;
    if ((int64_t)a.max_q * g.gqa > INT32_MAX / 2 ||
        (p.prompt && std::max(tiles * g.nkv, merges) >= kMostSegments) || segments + p.target >= kMostSegments)
      return fail("too many query rows in one call");
    if (p.bytes && (!workspace || workspace_bytes < p.bytes))
      return jacq::set_last_error(JACQ_KIVI_ENOMEM,
                                  "the workspace needs " + std::to_string(p.bytes) + " bytes, got " +
                                      std::to_string(workspace ? workspace_bytes : 0));
    uint8_t* ws = (uint8_t*)workspace;
    a.cus = device_cus();
    a.upto = INT32_MAX;
    if (p.few) {
      KiviAttendArgs few = a;
      if (p.prompt) few.upto = p.split;
      few.part_ml = (float*)(ws + p.few_ml);
      few.part_acc = (float*)(ws + p.few_acc);
      few.target = p.target;
      few.plan = p.planned ? (int32_t*)(ws + p.plan) : nullptr;
      few.rows = p.rows;
      few.row_blocks = p.row_blocks;
      if (int e = launched(jacq::launch_attend_few(g, few, p.nb, stream), "attention")) return e;
    }
    if (p.prompt) {
      a.above = p.split;
      a.part_ml = (float*)(ws + p.ml);
      a.part_acc = (float*)(ws + p.acc);
      a.slices = p.slices;
      a.tiles = (unsigned)tiles;
      a.merges = (unsigned)merges;
      a.slots = (int32_t*)(ws + p.slots);
      a.per_pass = p.per_pass;
      a.limit = p.passes == 1 ? p.per_pass : INT32_MAX;
      a.images = ws + p.images;
      a.poison = (uint64_t*)(ws + p.poison);
      return launched(jacq::launch_attend_prompt(g, a, p.passes, stream), "attention");
    }
    return JACQ_KIVI_OK;
  });
}

int jacq_kivi_read(const jacq_kivi_geometry* geo, const jacq_kivi_pool* pool, const int32_t* STARTS,
                   const int32_t* ENDS, const int32_t* BLOCK_TABLES, int32_t batch, int32_t total,
                   void* K, void* V, int32_t dtype, hipStream_t stream) {
  return guarded([&]() -> int {
    if (int e = check_geometry(geo)) return e;
    if (int e = check_pool(pool)) return e;
    if (int e = check_batch(batch)) return e;
    if (dtype < JACQ_KIVI_FP16 || dtype > JACQ_KIVI_FP32)
      return fail("values are read as fp16, bf16 or fp32");
    if (total < 0) return fail("negative number of tokens");
    if (batch == 0 || total == 0) return JACQ_KIVI_OK;
    if (!STARTS || !ENDS || (!BLOCK_TABLES && geo->max_pages_per_seq > 0) || !K || !V)
      return fail("a tensor pointer is null");
    if (!aligned({K, V}, 16) || !aligned({STARTS, ENDS, BLOCK_TABLES}, 4))
      return fail("K and V must be 16-byte aligned, tables 4-byte");
    if ((int64_t)geo->num_kv_heads * (total / jacq::kGroup + 2 * batch) >= 1 << 24)
      return fail("too many tokens in one read");
    return launched(jacq::launch_kivi_read(make_geo(*geo), read_pool(*pool), STARTS, ENDS,
                                           BLOCK_TABLES, batch, total, K, V, dtype, stream),
                    "read");
  });
}

}  // extern "C"
