// The code object of the kernels that work on a cache in pages: trees of drafted tokens, eviction.
#include "attend_tree.h"
#include "evict.h"

#define ATTEND_TREE(TYPE, T, DPAD, DUSE, NW, RT)                                                                            \
  extern "C" __global__ void __launch_bounds__(64 * NW, 1) attend_tree_##TYPE##_d##DUSE##_w##NW##_r##RT(TreeParams p) {    \
    attend::tree_body<T, DPAD, DUSE, NW, RT>(p);                                                                            \
  }
#define ATTEND_TREES(TYPE, T, DPAD, DUSE, NW) ATTEND_TREE(TYPE, T, DPAD, DUSE, NW, 1) ATTEND_TREE(TYPE, T, DPAD, DUSE, NW, 2)
ATTEND_TREES(bf16, bf16_t, 64, 64, 4)
ATTEND_TREES(bf16, bf16_t, 64, 64, 8)
ATTEND_TREES(bf16, bf16_t, 128, 128, 2)
ATTEND_TREES(bf16, bf16_t, 128, 128, 4)
ATTEND_TREES(f32, float, 64, 64, 2)
ATTEND_TREES(f32, float, 64, 64, 4)
#define ATTEND_TREE_ROWS(TYPE, T, DPAD, DUSE, BN, RT, OCC)                                                      \
  extern "C" __global__ void __launch_bounds__(256, OCC) attend_tree_##TYPE##_d##DUSE##_rows(TreeParams p) {       \
    attend::tree_rows_body<T, DPAD, DUSE, BN, RT>(p);                                                           \
  }
ATTEND_TREE_ROWS(bf16, bf16_t, 64, 64, 64, 2, 2)
ATTEND_TREE_ROWS(bf16, bf16_t, 128, 128, 32, 2, 2)
ATTEND_TREE_ROWS(bf16, bf16_t, 256, 256, 32, 1, 2)
ATTEND_TREE_ROWS(f32, float, 64, 64, 32, 2, 2)
ATTEND_TREE_ROWS(f32, float, 128, 128, 32, 1, 2)
ATTEND_TREE_ROWS(f32, float, 256, 256, 32, 1, 1)

extern "C" __global__ void __launch_bounds__(256) attend_tree_join_bf16(TreeParams p) { attend::tree_join_body<bf16_t>(p); }
extern "C" __global__ void __launch_bounds__(256) attend_tree_join_f32(TreeParams p) { attend::tree_join_body<float>(p); }

extern "C" __global__ void __launch_bounds__(1024) evict_select(EvictParams p) { attend::evict_select_body(p); }
extern "C" __global__ void __launch_bounds__(1024) evict_whole_bf16(EvictParams p) { attend::evict_whole_body(p, 2); }
extern "C" __global__ void __launch_bounds__(1024) evict_whole_f32(EvictParams p) { attend::evict_whole_body(p, 4); }
extern "C" __global__ void __launch_bounds__(256) evict_gather_bf16(EvictParams p) { attend::evict_gather_body(p, 2); }
extern "C" __global__ void __launch_bounds__(256) evict_gather_f32(EvictParams p) { attend::evict_gather_body(p, 4); }
