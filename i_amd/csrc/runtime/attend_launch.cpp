// Entry points of include/i_attend.h: checks of arguments, choice of kernels, launches.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "../../../include/i_attend.h"
#include "../kernels/attend_params.h"
#include "tree_checks.h"

namespace {

using namespace ihip::host;

// columns that the kernel for a head size works on
int columns(int64_t d, bool with_96) { return d <= 64 ? 64 : with_96 && d <= 96 ? 96 : d <= 128 ? 128 : 256; }

struct Plan {
  AttendParams p{};
  bool empty = false;  // nothing to compute (no sequence or no query)
};

Err plan_of(const i_attend_problem* a, Plan& plan) {
  if (!a) return "problem is missing";
  if (Err e = check_common(a->dtype, a->b, a->hq, a->hkv, a->d, a->scale, a->cap); !e.empty()) return e;
  if (Err e = check_extent("nq", a->nq); !e.empty()) return e;
  if (Err e = check_extent("nk", a->nk); !e.empty()) return e;
  if (a->causal != 0 && a->causal != 1) return "causal must be 0 or 1";
  AttendParams& p = plan.p;
  p.first = a->first;
  p.last = a->last;
  p.slopes = a->slopes;
  p.scale = (float)a->scale;
  p.cap = (float)a->cap;
  p.shift = (int32_t)(a->nk - a->nq);
  p.causal = (uint32_t)a->causal;
  p.b = (uint32_t)a->b;
  p.hq = (uint32_t)a->hq;
  p.hkv = (uint32_t)a->hkv;
  p.group = (uint32_t)(a->hq / a->hkv);
  p.nq = (uint32_t)a->nq;
  p.nk = (uint32_t)a->nk;
  p.d = (uint32_t)a->d;
  plan.empty = a->b == 0 || a->nq == 0;
  return {};
}

// A grid of `groups` x `tiles` that xcd_map deals out: whole runs for each of the 8 XCDs.
int64_t xcd_grid(int64_t groups, int64_t tiles) { return up(groups * tiles, 8); }

// Workgroups per key head of a kernel that walks keys, of which `slots` fit the chip at once: whole rounds of them, and no more than
// there are tiles of queries to walk, whatever a mask leaves of those.  A tile each is worth the partial results and their join: of 16 shapes from
// 3 heads of 257 to 32 of 2048, causal, windows, documents and whole, no gradient takes longer than with a half, a quarter or an eighth as
// many shares by more than 3 %, and no weights by more than 6 % (but f32, 4 x 4 x 333 x 128, documents: 18.4 us, with half as many
// 15.7).  bf16 gradients, us a call with as many, a quarter, an eighth: 3 x 257 x 64, a window 24.3, 26.1, 36.8; 8 x 777 x 64,
// a window 32.6, 35.0, 36.8; 4 x 4 x 333 x 128, documents 37.6, 39.3, 44.2;  f32: 3 x 257 x 64, causal 30.7, 39.3, 51.7; 8 x 777 x 64,
// causal 69.1, 69.1, 73.9;  f32 weights: 4 query heads of one key head of 512 x 128, causal 15.8, 20.6, 26.2.
int64_t key_shares(const AttendParams& p, int64_t key_tiles, int64_t query_tile, int64_t slots) {
  const int64_t heads = (int64_t)p.b * p.hkv, all = key_tiles * p.group * ceil_div(p.nq, query_tile);
  const int64_t most = std::max<int64_t>(1, all);
  if (heads >= slots) return 1;
  // one round, or two where heads do not divide it (96 heads on 256 slots: 5 shares fill two rounds to 94 %, 2 one to 75 %)
  const int64_t one = slots / heads, two = 2 * slots / heads;
  return std::min(most, one * heads * 10 >= slots * 9 ? one : two);
}

struct KeysShape {
  int tile, query_tile;  // keys a workgroup, rows of a query tile
  int slots = 256;       // workgroups that fit the chip at once
};
// (the template arguments of attend_grad_keys_* and attend_weights_*)
KeysShape gradient_keys(int64_t dtype, int cols) {
  if (dtype == I_DTYPE_BF16) return cols == 256 ? KeysShape{64, 32} : KeysShape{128, 64};
  return cols == 64 ? KeysShape{128, 32} : KeysShape{64, 32};
}
KeysShape weight_keys(int64_t dtype, int cols) {
  if (dtype == I_DTYPE_BF16) return cols == 256 ? KeysShape{128, 32, 512} : KeysShape{128, 64, 768};
  return cols == 256 ? KeysShape{64, 32, 256} : cols == 64 ? KeysShape{128, 32, 768} : KeysShape{128, 32, 512};
}
// (the plan counts the tiles of a key head in 32 bits, whatever the mask leaves of them)
Err check_work(const AttendParams& p, const KeysShape& shape) {
  const int64_t pairs = ceil_div(p.nk, shape.tile) * ceil_div(p.nq, shape.query_tile);
  if (pairs > kMaxGrid / p.group) return "a key head has 2^31 tiles of keys and queries or more";
  return {};
}
// (wavefronts whose tiles are their own: attend_fwd_few_*, attend_grad_queries_few_*, half as many attend_tree_*_r<n>)
int private_waves(int64_t dtype, int cols) {
  const int row_bytes = cols * (int)element_bytes(dtype);
  return row_bytes == 128 ? 8 : row_bytes == 256 ? 4 : row_bytes == 512 ? 2 : 1;
}
// How the queries are dealt out, by the number of 128-query tiles of all heads (times of bf16, d = 128, causal, 16 heads; forward,
// queries' gradient in us):
//   Few     16 a workgroup, whose wavefronts share out the keys.  16 tiles: few 9.5, 5.9; halves 9.3, 8.2.  32: few 9.2, 7.1; halves 9.3,
//           10.5.  64: few 17, 17.5; halves 12, 15.  (f32: 32 tiles: few 19, 21; halves 25.5, 33.  64: few 52, 63; halves 44, 58)
//   Halves  64 a workgroup of twice the wavefronts, half of the keys of a tile each.  128: halves 19, 25; whole 29.5, 44.  256: halves 44, 52; whole
//           53, 83 (not causal 49, 86 and 54, 84; f32 176, 243 and 281, 418).  1024: halves 322, 643; whole 278, 477.  In between it depends on the
//           mask (512 tiles, causal: halves 96, 173; whole 127, 209; not causal: halves 165, 314; whole 136, 230; documents of 400: halves
//           31.5, 50; whole 27, 37.5)
//   Whole   64 or 128 a workgroup
// The halves' tiles of 64 keys of 256 f32 columns do not fit the LDS.
enum class Queries { Few, Halves, Whole };
Queries queries_dealt(const i_attend_problem* a, int cols) {
  const int64_t tiles = a->b * a->hq * ceil_div(a->nq, 128);
  if (tiles < 64) return Queries::Few;
  return tiles <= 256 && !(a->dtype == I_DTYPE_F32 && cols == 256) ? Queries::Halves : Queries::Whole;
}
int forward_rows(int64_t dtype, int cols) { return dtype == I_DTYPE_F32 && cols == 256 ? 64 : 128; }
int gradient_rows(int64_t dtype, int cols) { return cols == 256 || (dtype == I_DTYPE_F32 && cols == 128) ? 64 : 128; }

// A kernel over tiles of queries.  rows_of: a workgroup's where they are dealt out whole.
Err run_queries(const std::string& kernel, const i_attend_problem* a, int (*rows_of)(int64_t, int), ihip::CodeObject object, AttendParams& p, hipStream_t stream) {
  const int padded = columns(a->d, false), cols = columns(a->d, true);
  const Queries dealt = queries_dealt(a, cols);
  const int rows = dealt == Queries::Few ? 16 : dealt == Queries::Halves ? 64 : rows_of(a->dtype, cols);
  const int threads = dealt == Queries::Few ? 64 * private_waves(a->dtype, padded) : dealt == Queries::Halves ? 512 : 256;
  const std::string name = kernel + (dealt == Queries::Few ? "few_" : dealt == Queries::Halves ? "halves_" : "") + type_name(a->dtype) + "_d" + std::to_string(dealt == Queries::Few ? padded : cols);
  p.tiles = (uint32_t)ceil_div(a->nq, rows);
  return run(name, object, xcd_grid(a->b * a->hq, p.tiles), threads, p, stream);
}

Err forward(const i_attend_problem* a, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* v, const i_attend_tensor* o,
            float* lse, hipStream_t stream) {
  Plan plan;
  if (Err e = plan_of(a, plan); !e.empty()) return e;
  if (plan.empty) return {};
  AttendParams& p = plan.p;
  for (auto [name, t] : {std::pair{"q", q}, {"o", o}})
    if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  if (a->nk > 0)
    for (auto [name, t] : {std::pair{"k", k}, {"v", v}})
      if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  p.q = operand(q);
  p.k = operand(k);
  p.v = operand(v);
  p.o = operand(o);
  p.lse = lse;
  return run_queries("attend_fwd_", a, forward_rows, ihip::CodeObject::AttendForward, p, stream);
}

// The division of the work on keys: key tiles of `shape`, `shares` workgroups a key head.
void divide_keys(AttendParams& p, const KeysShape& shape, int64_t shares, int* plan) {
  p.tiles = (uint32_t)ceil_div(p.nk, shape.tile);
  p.tile_keys = (uint32_t)shape.tile;
  p.query_rows = (uint32_t)shape.query_tile;
  p.shares = (uint32_t)shares;
  p.plan = plan;
}

struct BackwardScratch {
  float* rows;
  char* spans;
  float *partial_k, *partial_v;
  int* plan;
  int64_t shares;
  size_t bytes;
};
BackwardScratch backward_scratch(const AttendParams& p, int64_t dtype, char* base) {
  Carver c{base};
  BackwardScratch s{};
  const KeysShape shape = gradient_keys(dtype, columns(p.d, true));
  s.rows = c.take<float>((int64_t)p.b * p.hq * up(p.nq, 64) * 2);
  if (p.first || p.last) s.spans = c.take<char>((int64_t)p.b * ceil_div(p.nq, 64) * kSpanRecord);
  const int64_t tiles = ceil_div(p.nk, shape.tile);
  s.shares = key_shares(p, tiles, shape.query_tile, shape.slots);
  s.plan = c.take<int>(p.b * (2 * tiles + 1));
  if (s.shares > 1) {
    const int64_t partial = (int64_t)p.b * p.hkv * s.shares * 2 * shape.tile * p.d;
    s.partial_k = c.take<float>(partial);
    s.partial_v = c.take<float>(partial);
  }
  s.bytes = c.at;
  return s;
}

// `rows_each`: rows of a workgroup of the kernel
Err prepare(const std::string& name, int64_t rows_each, const AttendParams& p, hipStream_t stream) {
  const int64_t blocks = p.b + ceil_div((int64_t)p.b * p.hq * up(p.nq, 64), rows_each) + (p.spans ? ceil_div((int64_t)p.b * ceil_div(p.nq, 64), 4) : 0);
  return run(name, ihip::CodeObject::AttendBackward, blocks, 256, p, stream);
}

Err backward(const i_attend_problem* a, const i_attend_tensor* go, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* v,
             const i_attend_tensor* o, const float* lse, const i_attend_tensor* gq, const i_attend_tensor* gk, const i_attend_tensor* gv,
             void* workspace, size_t workspace_bytes, hipStream_t stream) {
  Plan plan;
  if (Err e = plan_of(a, plan); !e.empty()) return e;
  AttendParams& p = plan.p;
  if (a->b == 0) return {};
  if (a->nq > 0) {
    for (auto [name, t] : {std::pair{"grad_o", go}, {"q", q}, {"o", o}, {"grad_q", gq}})
      if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
    if (!lse) return "lse: null device pointer";
  }
  if (a->nk > 0)
    for (auto [name, t] : {std::pair{"k", k}, {"v", v}, {"grad_k", gk}, {"grad_v", gv}})
      if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  if (Err e = check_work(p, gradient_keys(a->dtype, columns(a->d, true))); !e.empty()) return e;
  const BackwardScratch s = backward_scratch(p, a->dtype, (char*)workspace);
  if (Err e = check_workspace(workspace, workspace_bytes, s.bytes); !e.empty()) return e;
  p.q = operand(q);
  p.k = operand(k);
  p.v = operand(v);
  p.o = operand(o);
  p.grad_o = operand(go);
  p.grad_q = operand(gq);
  p.grad_k = operand(gk);
  p.grad_v = operand(gv);
  p.lse = const_cast<float*>(lse);
  p.rows = s.rows;
  p.spans = s.spans;
  p.partial_k = s.partial_k;
  p.partial_v = s.partial_v;
  const int cols = columns(a->d, true);
  const std::string suffix = std::string(type_name(a->dtype)) + "_d" + std::to_string(cols);
  divide_keys(p, gradient_keys(a->dtype, cols), s.shares, s.plan);
  if (Err e = prepare(std::string("attend_prepare_") + type_name(a->dtype), 16, p, stream); !e.empty()) return e;
  if (a->nq > 0) {
    AttendParams of_q = p;
    if (Err e = run_queries("attend_grad_queries_", a, gradient_rows, ihip::CodeObject::AttendBackward, of_q, stream); !e.empty()) return e;
  }
  if (a->nk == 0) return {};
  if (Err e = run("attend_grad_keys_" + suffix, ihip::CodeObject::AttendBackward, xcd_grid(a->b * a->hkv, p.shares), 256, p, stream); !e.empty()) return e;
  if (p.shares == 1) return {};
  return run(std::string("attend_join_gradients_") + type_name(a->dtype), ihip::CodeObject::AttendBackward, a->b * a->hkv * p.tiles, 256, p, stream, 16);
}

struct WeightsScratch {
  float* rows;
  char* spans;
  float* partial;
  int* plan;
  int64_t shares;
  size_t bytes;
};
WeightsScratch weights_scratch(const AttendParams& p, int64_t dtype, char* base) {
  Carver c{base};
  WeightsScratch s{};
  const KeysShape shape = weight_keys(dtype, columns(p.d, true));
  s.rows = c.take<float>((int64_t)p.b * p.hq * up(p.nq, 64) * 2);
  if (p.first || p.last) s.spans = c.take<char>((int64_t)p.b * ceil_div(p.nq, 64) * kSpanRecord);
  const int64_t tiles = ceil_div(p.nk, shape.tile);
  s.shares = key_shares(p, tiles, shape.query_tile, shape.slots);
  s.plan = c.take<int>(p.b * (2 * tiles + 1));
  if (s.shares > 1) s.partial = c.take<float>((int64_t)p.b * p.hkv * s.shares * 2 * shape.tile);
  s.bytes = c.at;
  return s;
}

Err weights(const i_attend_problem* a, const i_attend_tensor* q, const i_attend_tensor* k, const float* lse, const float* weights_in,
            float* weights_out, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  Plan plan;
  if (Err e = plan_of(a, plan); !e.empty()) return e;
  AttendParams& p = plan.p;
  if (a->b == 0 || a->nk == 0) return {};
  if (a->nq > 0) {
    if (Err e = check_tensor("q", q, a->dtype); !e.empty()) return e;
    if (!lse) return "lse: null device pointer";
  }
  if (Err e = check_tensor("k", k, a->dtype); !e.empty()) return e;
  if (!weights_out) return "weights_out: null device pointer";
  if (Err e = check_work(p, weight_keys(a->dtype, columns(a->d, true))); !e.empty()) return e;
  const WeightsScratch s = weights_scratch(p, a->dtype, (char*)workspace);
  if (Err e = check_workspace(workspace, workspace_bytes, s.bytes); !e.empty()) return e;
  p.q = operand(q);
  p.k = operand(k);
  p.lse = const_cast<float*>(lse);
  p.rows = s.rows;
  p.spans = s.spans;
  p.partial_k = s.partial;
  p.weights_in = weights_in;
  p.weights_out = weights_out;
  const int cols = columns(a->d, true);
  divide_keys(p, weight_keys(a->dtype, cols), s.shares, s.plan);
  if (Err e = prepare("attend_prepare_weights", 256, p, stream); !e.empty()) return e;
  const std::string name = std::string("attend_weights_") + type_name(a->dtype) + "_d" + std::to_string(cols);
  if (Err e = run(name, ihip::CodeObject::AttendBackward, xcd_grid(a->b * a->hkv, p.shares), 256, p, stream); !e.empty()) return e;
  if (p.shares == 1) return {};
  return run("attend_join_weights", ihip::CodeObject::AttendBackward, a->b * a->hkv * p.tiles, 256, p, stream);
}

Err cache_of(const char* name, const i_attend_cache* c, int64_t dtype, int64_t b, int64_t slots, AttendCache& out) {
  if (!c) return std::string(name) + " is missing";
  const int64_t e = (int64_t)element_bytes(dtype);
  if (c->page < 1 || c->page > kMaxExtent) return std::string(name) + ": page size must be 1 .. 2^30";
  if (c->pages < 0 || c->pages > kMaxExtent) return std::string(name) + ": pages must be 0 .. 2^30";
  const int64_t per = c->table ? c->table_stride : 1;
  if (slots > 0 && c->pages < 1) return std::string(name) + " has no pages";
  if (c->table_stride < 0) return std::string(name) + ": negative table stride";
  if (!c->table && b > c->pages) return std::string(name) + ": without a table every sequence needs a page of its own";
  if (per < ceil_div(slots, c->page)) return std::string(name) + ": " + std::to_string(slots) + " slots do not fit " + std::to_string(per) + " pages of " + std::to_string(c->page);
  if (slots > 0) {
    if (!c->k || !c->v) return std::string(name) + ": null device pointer";
    if ((uintptr_t)c->k % 16 != 0 || (uintptr_t)c->v % 16 != 0) return std::string(name) + " must start on a 16-byte boundary";
  }
  for (int64_t s : {c->k_stride_page, c->k_stride_head, c->k_stride_slot, c->v_stride_page, c->v_stride_head, c->v_stride_slot}) {
    if (s < 0) return std::string(name) + ": negative strides are not supported";
    if (s * e % 16 != 0) return std::string(name) + ": strides must be multiples of 16 bytes";
  }
  out.k = c->k;
  out.v = c->v;
  out.k_page = c->k_stride_page;
  out.k_head = c->k_stride_head;
  out.k_slot = c->k_stride_slot;
  out.v_page = c->v_stride_page;
  out.v_head = c->v_stride_head;
  out.v_slot = c->v_stride_slot;
  out.table = c->table;
  out.table_stride = c->table_stride;
  out.page = (uint32_t)c->page;
  out.pages = (uint32_t)c->pages;
  return {};
}

struct TreePlan {
  TreeParams p{};
  int row_blocks = 1;   // of 16 rows, per wavefront
  bool shared = false;  // dealt out to a workgroup's wavefronts
  int waves = 4;
  int cols = 64;
  size_t bytes = 0;
};

Err tree_plan(const i_attend_tree_problem* a, char* base, TreePlan& plan) {
  TreeParams& p = plan.p;
  if (Err e = tree_problem(a, p); !e.empty()) return e;
  plan.cols = columns(a->d, false);
  // Up to 32 rows stay with each wavefront, which walk keys of their own; more are dealt out to the wavefronts of a workgroup, which
  // share their tiles (8 x 8 heads of 4096 bf16 keys, 128 columns: 4 rows 34 us a call, shared 39; 24 rows of 64 columns 29 and 30; 32 rows
  // 45 and 42, but 38 and 42 for 16 x 2000).  Rows of 512 bytes and more leave LDS for a wavefront with tiles of its own or two, and
  // share them always (256 bf16 columns, 8 rows: 67 us, shared 58; 32 rows: 104 and 61; f32, 128 columns, 1 row: 83 and 69).
  const int row_bytes = plan.cols * (int)element_bytes(a->dtype);
  plan.shared = p.rows > 32 || row_bytes >= 512;
  int64_t slots = plan.cols == 256 && a->dtype == I_DTYPE_F32 ? 256 : 512;  // workgroups that the chip holds at once
  if (!plan.shared) {
    plan.row_blocks = p.rows <= 16 ? 1 : 2;
    plan.waves = private_waves(a->dtype, plan.cols) / 2;
    p.row_tiles = 1;
    p.unit = (uint32_t)(32 * plan.waves);
  } else {
    plan.row_blocks = row_bytes <= 256 ? 2 : 1;
    plan.waves = 4;
    p.row_tiles = (uint32_t)ceil_div(p.rows, 64 * plan.row_blocks);
    p.unit = a->dtype == I_DTYPE_BF16 && plan.cols <= 64 ? 64 : 32;
  }
  const int64_t heads = a->b * a->hkv, units = ceil_div(a->max_length, p.unit);
  if (heads * units > (1ll << 31)) return "the cache has more than 2^31 tiles of keys";
  if (heads * p.rows > kMaxGrid) return "the drafted tokens have 2^31 rows (of all sequences and query heads) or more";
  // Short caches: a workgroup has a head's keys to itself, which saves the second launch.  Up to 8 units of bf16 (64 sequences of 500
  // keys, 32 x 128 heads: 20 us a call against 26 in runs), or what takes as long with f32 products (128 columns, 200 keys, 7 units: 33
  // against 17).  Where the chip holds all heads at once and the wavefronts have tiles of their own, twice the wavefronts and twice the keys (8
  // heads of 64 columns, f32: 200 keys 12.7 against 14.5 with as many wavefronts, 500 keys 12.8 against 16.8 in runs; bf16, 2000 keys: 13
  // against 16; 32 x 8 heads of 1000 x 128: 20.5 against 25).
  const bool few_heads = heads <= 256 && !plan.shared;
  p.whole_heads = units * (a->dtype == I_DTYPE_F32 ? plan.cols / 32 : 1) <= (few_heads ? 16 : 8);
  if (p.whole_heads && few_heads) plan.waves *= 2;
  p.runs = (uint32_t)(p.whole_heads ? heads : std::max<int64_t>(1, std::min(heads * units, slots / p.row_tiles)));
  p.score_stride = (uint32_t)(units * p.unit);
  Carver c{base};
  const bool weights = a->weights_out && p.counted_nodes > 0;
  if (!p.whole_heads) {
    p.partial_o = c.take<float>((int64_t)p.runs * 2 * p.rows * p.d);
    p.partial_lse = c.take<float>((int64_t)p.runs * 2 * p.rows);
  }
  if (!p.whole_heads || weights) p.head_runs = c.take<int>(heads * 2);
  if (weights) p.head_lse = c.take<float>(heads * p.rows);
  if (weights) p.scores = c.take<float>(heads * p.group * p.counted_nodes * p.score_stride);
  plan.bytes = c.at;
  return {};
}

Err tree(const i_attend_tree_problem* a, const i_attend_tensor* q, const i_attend_cache* cache, const i_attend_tensor* o, float* lse,
         void* workspace, size_t workspace_bytes, hipStream_t stream) {
  TreePlan plan;
  if (Err e = tree_plan(a, (char*)workspace, plan); !e.empty()) return e;
  TreeParams& p = plan.p;
  if (a->b == 0) return {};
  for (auto [name, t] : {std::pair{"q", q}, {"o", o}})
    if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  if (Err e = cache_of("cache", cache, a->dtype, a->b, a->max_length, p.cache); !e.empty()) return e;
  if (Err e = check_tree_arrays(a); !e.empty()) return e;
  if (Err e = check_workspace(workspace, workspace_bytes, plan.bytes); !e.empty()) return e;
  p.q = operand(q);
  p.o = operand(o);
  p.lse = lse;
  const std::string name = std::string("attend_tree_") + type_name(a->dtype) + "_d" + std::to_string(plan.cols) + (plan.shared ? "_rows" : "_w" + std::to_string(plan.waves) + "_r" + std::to_string(plan.row_blocks));
  const Divider pages(p.cache.page);
  p.page_magic = pages.magic;
  p.page_shift = pages.shift;
  const int64_t grid = plan.shared ? up(p.runs, 8) * p.row_tiles : p.runs;
  if (Err e = run(name, ihip::CodeObject::AttendCache, grid, 64 * plan.waves, p, stream); !e.empty()) return e;
  const int64_t join = p.whole_heads ? 0 : ceil_div((int64_t)p.b * p.hkv * p.rows, 4);
  const int64_t weigh = a->weights_out ? (int64_t)p.b * p.hkv * ceil_div(p.max_length, 1024) : 0;
  if (join + weigh == 0) return {};
  return run(std::string("attend_tree_join_") + type_name(a->dtype), ihip::CodeObject::AttendCache, join + weigh, 256, p, stream);
}

Err evict_plan(const i_evict_problem* a, char* base, EvictParams& p, size_t& bytes) {
  if (!a) return "problem is missing";
  if (Err e = check_common(a->dtype, a->b, a->hkv, a->hkv, a->d, 1.0, 0.0); !e.empty()) return e;
  if (a->keep < 1 || a->keep > kMaxExtent) return "keep must be 1 .. 2^30, not " + std::to_string(a->keep);
  if (a->recent < 0 || a->recent > a->keep) return "recent must be 0 .. keep, not " + std::to_string(a->recent);
  if (Err e = check_extent("max_length", a->max_length); !e.empty()) return e;
  Carver c{base};
  p.chosen = c.take<int>(a->b * a->hkv * a->keep);
  bytes = c.at;
  return {};
}

// whether two arrays of 4-byte elements share memory (a null one does not)
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && na > 0 && nb > 0 && x < y + 4 * (uintptr_t)nb && y < x + 4 * (uintptr_t)na;
}

Err evict(const i_evict_problem* a, const i_attend_cache* from, const i_attend_cache* to, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  EvictParams p{};
  size_t bytes = 0;
  if (Err e = evict_plan(a, (char*)workspace, p, bytes); !e.empty()) return e;
  if (a->b == 0) return {};
  const int64_t most = std::min(a->keep, a->max_length);  // entries that may stay
  if (Err e = cache_of("from", from, a->dtype, a->b, a->max_length, p.from); !e.empty()) return e;
  if (Err e = cache_of("to", to, a->dtype, a->b, most, p.to); !e.empty()) return e;
  if (!a->lengths || !a->lengths_out || !a->weights || !a->weights_out || !a->positions_out) return "lengths, weights or an output: null device pointer";
  if (a->weights_stride < a->max_length) return "weights must have max_length entries a head";
  if (a->positions && a->positions_stride < a->max_length) return "positions must have max_length entries a head";
  if (a->out_stride < most) return "the outputs must have room for what stays";
  const int64_t heads = a->b * a->hkv;
  auto entries = [&](int64_t stride) { return heads * std::min(stride, kMaxExtent); };
  if (overlap(a->lengths, a->b, a->lengths_out, a->b)) return "the old lengths and the new ones share memory";
  if (overlap(a->weights, entries(a->weights_stride), a->weights_out, entries(a->out_stride))) return "the old weights and the new ones share memory";
  if (overlap(a->positions, entries(a->positions_stride), a->positions_out, entries(a->out_stride))) return "the old positions and the new ones share memory";
  if (Err e = check_workspace(workspace, workspace_bytes, bytes); !e.empty()) return e;
  p.lengths = a->lengths;
  p.weights = a->weights;
  p.positions = a->positions;
  p.weights_stride = a->weights_stride;
  p.positions_stride = a->positions_stride;
  p.weights_out = a->weights_out;
  p.positions_out = a->positions_out;
  p.lengths_out = a->lengths_out;
  p.out_stride = a->out_stride;
  p.b = (uint32_t)a->b;
  p.hkv = (uint32_t)a->hkv;
  p.d = (uint32_t)a->d;
  p.keep = (uint32_t)a->keep;
  p.recent = (uint32_t)a->recent;
  p.max_length = (uint32_t)a->max_length;
  p.row_bytes = (uint32_t)(a->d * (int64_t)element_bytes(a->dtype));
  p.tiles = (uint32_t)ceil_div(most, 64);
  // Few rows are moved by the workgroup that selected them, which saves a launch and moves 64 rows after another.  8 heads and 128, one
  // launch and two in us a call (range over caches of 300 .. 16000 slots):  128 rows of 1024 bytes 15.2 .. 28.2 and 17.1 .. 28.9, of 128 bytes
  // 14.4 .. 19.5 and 16.8 .. 19.5;  256 rows of 256 bytes, up to 4000 slots 14.4 .. 18.3 and 16.8 .. 17.1, 16000 slots 22.2 .. 24.8
  // and 19.6 .. 23.4;  256 rows of 1024 bytes 21.0 .. 39.0 and 17.1 .. 38.9;  384 rows of 256 bytes 17.2 .. 29.2 and 16.9 .. 26.4.
  if (most <= 128 || (most <= 256 && p.row_bytes <= 256 && p.max_length <= 4096))
    return run(std::string("evict_whole_") + type_name(a->dtype), ihip::CodeObject::AttendCache, a->b * a->hkv, 1024, p, stream);
  if (Err e = run("evict_select", ihip::CodeObject::AttendCache, a->b * a->hkv, 1024, p, stream); !e.empty()) return e;
  return run(std::string("evict_gather_") + type_name(a->dtype), ihip::CodeObject::AttendCache, a->b * a->hkv * p.tiles, 256, p, stream);
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

int i_attend(const i_attend_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* v,
             const i_attend_tensor* o, float* lse, void* stream) {
  return guarded("attention", [&] { return forward(problem, q, k, v, o, lse, (hipStream_t)stream); });
}

size_t i_attend_backward_workspace(const i_attend_problem* problem) {
  size_t bytes = (size_t)-1;
  guarded("attention_backward", [&] {
    Plan plan;
    if (Err e = plan_of(problem, plan); !e.empty()) return e;
    if (Err e = check_work(plan.p, gradient_keys(problem->dtype, columns(problem->d, true))); !e.empty()) return e;
    bytes = problem->b == 0 ? 0 : backward_scratch(plan.p, problem->dtype, nullptr).bytes;
    return Err{};
  });
  return bytes;
}

int i_attend_backward(const i_attend_problem* problem, const i_attend_tensor* grad_o, const i_attend_tensor* q, const i_attend_tensor* k,
                      const i_attend_tensor* v, const i_attend_tensor* o, const float* lse, const i_attend_tensor* grad_q,
                      const i_attend_tensor* grad_k, const i_attend_tensor* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("attention_backward", [&] {
    return backward(problem, grad_o, q, k, v, o, lse, grad_q, grad_k, grad_v, workspace, workspace_bytes, (hipStream_t)stream);
  });
}

size_t i_attend_weights_workspace(const i_attend_problem* problem) {
  size_t bytes = (size_t)-1;
  guarded("key_weights", [&] {
    Plan plan;
    if (Err e = plan_of(problem, plan); !e.empty()) return e;
    if (Err e = check_work(plan.p, weight_keys(problem->dtype, columns(problem->d, true))); !e.empty()) return e;
    bytes = problem->b == 0 || problem->nk == 0 ? 0 : weights_scratch(plan.p, problem->dtype, nullptr).bytes;
    return Err{};
  });
  return bytes;
}

int i_attend_weights(const i_attend_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const float* lse,
                     const float* weights_in, float* weights_out, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("key_weights", [&] {
    return weights(problem, q, k, lse, weights_in, weights_out, workspace, workspace_bytes, (hipStream_t)stream);
  });
}

size_t i_attend_tree_workspace(const i_attend_tree_problem* problem) {
  size_t bytes = (size_t)-1;
  guarded("tree_attention", [&] {
    TreePlan plan;
    if (Err e = tree_plan(problem, nullptr, plan); !e.empty()) return e;
    bytes = problem->b == 0 ? 0 : plan.bytes;
    return Err{};
  });
  return bytes;
}

int i_attend_tree(const i_attend_tree_problem* problem, const i_attend_tensor* q, const i_attend_cache* cache, const i_attend_tensor* o,
                  float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("tree_attention", [&] { return tree(problem, q, cache, o, lse, workspace, workspace_bytes, (hipStream_t)stream); });
}

size_t i_evict_workspace(const i_evict_problem* problem) {
  size_t bytes = (size_t)-1;
  guarded("evict", [&] {
    EvictParams p{};
    size_t needed = 0;
    if (Err e = evict_plan(problem, nullptr, p, needed); !e.empty()) return e;
    bytes = problem->b == 0 ? 0 : needed;
    return Err{};
  });
  return bytes;
}

int i_evict(const i_evict_problem* problem, const i_attend_cache* from, const i_attend_cache* to, void* workspace, size_t workspace_bytes,
            void* stream) {
  return guarded("evict", [&] { return evict(problem, from, to, workspace, workspace_bytes, (hipStream_t)stream); });
}

}  // extern "C"
#pragma GCC visibility pop
