// Entry points of include/i_quantised.h: checks of arguments, choice of kernels, launches.
#include "../../../include/i_quantised.h"

#include <utility>

#include "../kernels/quantised_params.h"
#include "tree_checks.h"

namespace {

using namespace ihip::host;

int64_t blocks_of(int64_t d) { return ceil_div(d, 32); }

Err check_bits(int64_t bits) {
  if (bits != 4 && bits != 8) return "bits must be 4 or 8, not " + std::to_string(bits);
  return {};
}

Err side_of(const char* name, void* codes, void* scales, const int64_t (&strides)[6], bool read, QuantisedSide& out) {
  if (read) {
    if (!codes || !scales) return std::string(name) + ": null device pointer";
    if ((uintptr_t)codes % 16 != 0) return std::string(name) + " must start on a 16-byte boundary";
  }
  for (int n = 0; n < 6; ++n) {
    if (strides[n] < 0) return std::string(name) + ": negative strides are not supported";
    if (n < 3 && strides[n] % 16 != 0) return std::string(name) + ": strides must be multiples of 16 bytes";
    // (16 rows are addressed from the first of them in 32 bits)
    if (n % 3 == 2 && strides[n] >= (int64_t(1) << 25)) return std::string(name) + ": rows more than 32 MiB apart are not supported";
  }
  out = QuantisedSide{(uint8_t*)codes, (uint8_t*)scales, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5]};
  return {};
}

// pages that a sequence has
int64_t listed_of(const i_quantised_cache* c) { return !c->table ? 1 : c->listed > 0 ? c->listed : c->table_stride; }

// Checks the cache for b sequences of which `slots` slots are reached (0: none that the pages do not have).
Err cache_of(const i_quantised_cache* c, int64_t b, int64_t slots, QuantisedSide& k, QuantisedSide& v) {
  if (!c) return "cache is missing";
  if (Err e = check_bits(c->bits); !e.empty()) return e;
  if (c->page < 1 || c->page > kMaxExtent) return "cache: page size must be 1 .. 2^30";
  if (c->pages < 0 || c->pages > kMaxExtent) return "cache: pages must be 0 .. 2^30";
  if (c->table_stride < 0 || c->table_stride > kMaxExtent) return "cache: table stride must be 0 .. 2^30";
  if (c->listed < 0 || c->listed > kMaxExtent) return "cache: listed pages must be 0 .. 2^30";
  if (!c->table && b > c->pages) return "cache: without a table every sequence needs a page of its own";
  const int64_t per = listed_of(c);
  if (slots > 0 && c->pages < 1) return "cache has no pages";
  if (per < ceil_div(slots, c->page)) return "cache: " + std::to_string(slots) + " slots do not fit " + std::to_string(per) + " pages of " + std::to_string(c->page);
  const bool read = c->pages > 0;
  if (Err e = side_of("cache k", c->k, c->k_scales, {c->k_stride_page, c->k_stride_head, c->k_stride_slot, c->k_scales_stride_page, c->k_scales_stride_head, c->k_scales_stride_slot}, read, k); !e.empty()) return e;
  return side_of("cache v", c->v, c->v_scales, {c->v_stride_page, c->v_stride_head, c->v_stride_slot, c->v_scales_stride_page, c->v_scales_stride_head, c->v_scales_stride_slot}, read, v);
}

Err move(const char* kernel, const i_quantised_problem* a, const i_attend_tensor* k, const i_attend_tensor* v, const i_quantised_cache* cache, hipStream_t stream) {
  if (!a) return "problem is missing";
  if (Err e = check_common(a->dtype, a->b, a->hkv, a->hkv, a->d, 1.0, 0.0); !e.empty()) return e;
  if (Err e = check_extent("n", a->n); !e.empty()) return e;
  QuantisedMoveParams p{};
  if (Err e = cache_of(cache, a->b, 0, p.k_cache, p.v_cache); !e.empty()) return e;
  const int64_t tokens = a->b * a->n;
  if (tokens > kMaxExtent || tokens * a->hkv > kMaxExtent) return "more than 2^30 rows";
  if (tokens == 0) return {};
  for (auto [name, t] : {std::pair{"k", k}, {"v", v}})
    if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  p.k = operand(k);
  p.v = operand(v);
  p.table = cache->table;
  p.table_stride = cache->table_stride;
  p.first = a->first;
  p.counts = a->counts;
  p.page = (uint32_t)cache->page;
  p.pages = (uint32_t)cache->pages;
  const Divider page((uint32_t)cache->page), head((uint32_t)a->hkv), token((uint32_t)a->n);
  p.page_magic = page.magic;
  p.page_shift = page.shift;
  p.head_magic = head.magic;
  p.head_shift = head.shift;
  p.token_magic = token.magic;
  p.token_shift = token.shift;
  // (a cache without pages has no slot; slots are counted in 31 bits, more than any `first` reaches)
  p.slots = cache->pages == 0 ? 0 : (uint32_t)std::min<int64_t>(cache->page * listed_of(cache), 0x7fffffff);
  p.b = (uint32_t)a->b;
  p.hkv = (uint32_t)a->hkv;
  p.n = (uint32_t)a->n;
  p.d = (uint32_t)a->d;
  p.rows = (uint32_t)(tokens * a->hkv);
  const int64_t blocks = blocks_of(a->d);
  const int lanes = blocks <= 1 ? 4 : blocks <= 2 ? 8 : blocks <= 4 ? 16 : 32;
  const std::string name = std::string(kernel) + type_name(a->dtype) + "_b" + std::to_string(cache->bits) + "_l" + std::to_string(lanes);
  const int64_t workgroups = ceil_div((int64_t)p.rows * lanes, 256), across = int64_t(1) << kMoveAcross;
  return run(name, ihip::CodeObject::Quantised, std::min(workgroups, across), 256, p, stream, (unsigned)ceil_div(workgroups, across));
}

struct TreePlan {
  QuantisedTreeParams p{};
  int cols = 64;
  bool few = false;  // a wavefront's tiles are its own
  size_t bytes = 0;
};

Err tree_plan(const i_attend_tree_problem* a, int64_t bits, char* base, TreePlan& plan) {
  TreeParams& p = plan.p.tree;
  if (Err e = tree_problem(a, p); !e.empty()) return e;
  if (Err e = check_bits(bits); !e.empty()) return e;
  if (a->weights_in || a->weights_out) return "weights are not kept over a cache in few bits";
  plan.cols = a->d <= 64 ? 64 : a->d <= 128 ? 128 : 256;
  plan.few = p.rows <= 16;
  const bool f32 = a->dtype == I_DTYPE_F32;
  // workgroups that the chip holds at once
  const int64_t slots = 256 * (plan.few ? (plan.cols == 256 || (plan.cols == 128 && f32 && bits == 4) ? 1 : 2) : plan.cols == 256 ? (f32 ? 1 : 2) : f32 ? 2 : 3);
  p.row_tiles = plan.few ? 1 : (uint32_t)ceil_div(p.rows, 64);
  p.unit = plan.few ? (bits == 4 ? 256 : 128) : plan.cols <= 64 ? 64 : 32;
  const int64_t heads = a->b * a->hkv, units = ceil_div(a->max_length, p.unit);
  // Beginning with a head takes as long as this many units (32 sequences of up to 8192 keys, one token: us with 0, 1, 2, 3, 5 of them
  // 53.6, 49.0, 47.4, 46.9, 48.6;  trees of 48, 0, 1, 2, 4: 52.7, 51.8, 51.4, 50.4;  both of bf16, 4 bits, 128 columns: the other types, bits and
  // head sizes take them over).
  const int64_t begin_units = plan.few ? 2 : 4;
  if (heads * (units + begin_units) > (1ll << 31)) return "the cache has more than 2^31 tiles of keys";
  if (heads * p.rows > kMaxGrid) return "the drafted tokens have 2^31 rows (of all sequences and query heads) or more";
  // Short caches: a workgroup has a head's keys to itself, which saves the partial results and the second launch.  Up to 16 rows, us whole and
  // in runs: 8 heads of 1000 keys (4 units of 256) 15.6 and 17, of 2000 23.5 and 16; 256 heads of 1000 16.7 and 20, of 2000 26 and 23; 512 of
  // 2000 29 and 31.  More, units of 32: 64 rows of 64 heads of 250 keys 15 and 20, of 500 21 and 20, of 800 28 and 21; of 256 heads of 500
  // (17 units) 22.5 and 28, of 1000 37 and 32.
  p.whole_heads = units <= (plan.few ? (heads < 512 ? 4 : 8) : heads * p.row_tiles < 256 ? 16 : 24);
  // Else as many runs as the chip holds, but for 64 rows, whose partial results cost as much as the keys: a run's take about 8 bytes a column
  // at 4 TB/s, a unit 0.65 us (bf16, 4 bits, 128 columns, taken over for the rest), so that the sum is least at this many runs (64 heads of 1200
  // keys, 64 rows: 768 runs 37 us, 304 22).
  int64_t runs = std::min(heads * units, slots / p.row_tiles);
  if (!plan.few) runs = std::min(runs, std::max(std::min(heads, runs), (int64_t)std::sqrt((double)(heads * units) * 325000.0 / (double)(ceil_div(p.rows, p.row_tiles) * p.d))));
  p.runs = (uint32_t)(p.whole_heads ? heads : std::max<int64_t>(1, runs));
  if (up(p.runs, 8) * p.row_tiles * 256 > kMaxThreads || (!p.whole_heads && ceil_div(heads * p.rows, 4) * 256 > kMaxThreads))
    return "the drafted tokens have more rows than a launch";
  p.score_stride = 0;
  if (!p.whole_heads) p.begin_units = (uint32_t)begin_units;
  Carver c{base};
  if (!p.whole_heads) {
    p.partial_o = c.take<float>((int64_t)p.runs * 2 * p.rows * p.d);
    p.partial_lse = c.take<float>((int64_t)p.runs * 2 * p.rows);
    p.head_runs = c.take<int>(heads * 2);
  }
  plan.bytes = c.at;
  return {};
}

Err tree(const i_attend_tree_problem* a, const i_attend_tensor* q, const i_quantised_cache* cache, const i_attend_tensor* o, float* lse,
         void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!cache) return "cache is missing";
  TreePlan plan;
  if (Err e = tree_plan(a, cache->bits, (char*)workspace, plan); !e.empty()) return e;
  TreeParams& p = plan.p.tree;
  if (a->b == 0) return {};
  for (auto [name, t] : {std::pair{"q", q}, {"o", o}})
    if (Err e = check_tensor(name, t, a->dtype); !e.empty()) return e;
  if (Err e = cache_of(cache, a->b, a->max_length, plan.p.k, plan.p.v); !e.empty()) return e;
  if (Err e = check_tree_arrays(a); !e.empty()) return e;
  if (Err e = check_workspace(workspace, workspace_bytes, plan.bytes); !e.empty()) return e;
  p.q = operand(q);
  p.o = operand(o);
  p.lse = lse;
  p.cache.table = cache->table;
  p.cache.table_stride = cache->table_stride;
  p.cache.page = (uint32_t)cache->page;
  p.cache.pages = (uint32_t)cache->pages;
  const Divider page((uint32_t)cache->page);
  p.page_magic = page.magic;
  p.page_shift = page.shift;
  const std::string name = std::string("attend_quantised_") + type_name(a->dtype) + "_b" + std::to_string(cache->bits) + "_d" + std::to_string(plan.cols) + (plan.few ? "_few" : "_rows");
  if (Err e = run(name, ihip::CodeObject::Quantised, up(p.runs, 8) * p.row_tiles, 256, plan.p, stream); !e.empty()) return e;
  if (p.whole_heads) return {};
  const int64_t all_rows = (int64_t)p.b * p.hkv * p.rows;
  // A workgroup a row where heads have many runs each and rows are few, else a few lanes a row: us whole with that and with this for 4 heads of
  // 128 runs, 4 rows each 19.8 and 34.3;  32 of 16, 4 rows 18.6 and 19.5;  64 of 8, 16 rows 27.1 and 27.1;  32 of 8, 192 rows 59.8 and 57.3.
  const bool many = (int64_t)p.runs >= 8 * a->b * a->hkv && all_rows <= 2048;
  return run(std::string(many ? "attend_quantised_join_" : "attend_quantised_few_join_") + type_name(a->dtype) + "_d" + std::to_string(plan.cols),
             ihip::CodeObject::Quantised, many ? all_rows : ceil_div(all_rows * plan.cols, 1024), 256, p, stream);
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

int i_quantised_store(const i_quantised_problem* problem, const i_attend_tensor* k, const i_attend_tensor* v, const i_quantised_cache* cache, void* stream) {
  return guarded("store", [&] { return move("cache_store_", problem, k, v, cache, (hipStream_t)stream); });
}

int i_quantised_load(const i_quantised_problem* problem, const i_quantised_cache* cache, const i_attend_tensor* k, const i_attend_tensor* v, void* stream) {
  return guarded("load", [&] { return move("cache_load_", problem, k, v, cache, (hipStream_t)stream); });
}

size_t i_attend_quantised_workspace(const i_attend_tree_problem* problem, int64_t bits) {
  size_t bytes = (size_t)-1;
  guarded("tree_attention", [&] {
    TreePlan plan;
    if (Err e = tree_plan(problem, bits, nullptr, plan); !e.empty()) return e;
    bytes = problem->b == 0 ? 0 : plan.bytes;
    return Err{};
  });
  return bytes;
}

int i_attend_quantised(const i_attend_tree_problem* problem, const i_attend_tensor* q, const i_quantised_cache* cache, const i_attend_tensor* o,
                       float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("tree_attention", [&] { return tree(problem, q, cache, o, lse, workspace, workspace_bytes, (hipStream_t)stream); });
}

}  // extern "C"
#pragma GCC visibility pop
