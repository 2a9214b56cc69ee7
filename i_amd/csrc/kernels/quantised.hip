// The code object of a cache in 8 or 4 bits: writing, reading back, attention over it.
#include "attend_quantised.h"

#define CACHE_MOVE(TYPE, T, BITS, LPR)                                                                             \
  extern "C" __global__ void __launch_bounds__(256) cache_store_##TYPE##_b##BITS##_l##LPR(QuantisedMoveParams p) { \
    attend::store_body<T, BITS, LPR>(p);                                                                           \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(256) cache_load_##TYPE##_b##BITS##_l##LPR(QuantisedMoveParams p) {  \
    attend::load_body<T, BITS, LPR>(p);                                                                            \
  }
#define CACHE_MOVES(TYPE, T, BITS) CACHE_MOVE(TYPE, T, BITS, 4) CACHE_MOVE(TYPE, T, BITS, 8) CACHE_MOVE(TYPE, T, BITS, 16) CACHE_MOVE(TYPE, T, BITS, 32)
CACHE_MOVES(bf16, bf16_t, 4)
CACHE_MOVES(bf16, bf16_t, 8)
CACHE_MOVES(f32, float, 4)
CACHE_MOVES(f32, float, 8)

// (the last argument: workgroups that a compute unit holds, which the launcher counts on)
#define ATTEND_QUANTISED_ROWS(TYPE, T, BITS, DPAD, BN, OCC)                                                                          \
  extern "C" __global__ void __launch_bounds__(256, OCC) attend_quantised_##TYPE##_b##BITS##_d##DPAD##_rows(QuantisedTreeParams p) { \
    attend::quantised_rows_body<T, BITS, DPAD, BN>(p);                                                                               \
  }
#define ATTEND_QUANTISED_ALL_ROWS(BITS)                       \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 64, 64, 3)        \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 128, 32, 3)       \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 256, 32, 2)       \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 64, 64, 2)          \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 128, 32, 2)         \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 256, 32, 1)
ATTEND_QUANTISED_ALL_ROWS(4)
ATTEND_QUANTISED_ALL_ROWS(8)

#define ATTEND_QUANTISED_FEW(TYPE, T, BITS, DPAD, NW, OCC)                                                                                   \
  extern "C" __global__ void __launch_bounds__(64 * NW, OCC) attend_quantised_##TYPE##_b##BITS##_d##DPAD##_few(QuantisedTreeParams p) { \
    attend::quantised_few_body<T, BITS, DPAD, NW>(p);                                                                               \
  }
#define ATTEND_QUANTISED_FEWS(TYPE, T, BITS, OCC) \
  ATTEND_QUANTISED_FEW(TYPE, T, BITS, 64, 4, 2) ATTEND_QUANTISED_FEW(TYPE, T, BITS, 128, 4, OCC) ATTEND_QUANTISED_FEW(TYPE, T, BITS, 256, 4, 1)
ATTEND_QUANTISED_FEWS(bf16, bf16_t, 4, 2)
ATTEND_QUANTISED_FEWS(bf16, bf16_t, 8, 2)
ATTEND_QUANTISED_FEWS(f32, float, 4, 1)
ATTEND_QUANTISED_FEWS(f32, float, 8, 2)

#define ATTEND_QUANTISED_JOIN(TYPE, T, DPAD)                                                                                                             \
  extern "C" __global__ void __launch_bounds__(256) attend_quantised_few_join_##TYPE##_d##DPAD(TreeParams p) { attend::quantised_few_join_body<T, DPAD>(p); } \
  extern "C" __global__ void __launch_bounds__(256) attend_quantised_join_##TYPE##_d##DPAD(TreeParams p) { attend::quantised_join_body<T, DPAD>(p); }
ATTEND_QUANTISED_JOIN(bf16, bf16_t, 64)
ATTEND_QUANTISED_JOIN(bf16, bf16_t, 128)
ATTEND_QUANTISED_JOIN(bf16, bf16_t, 256)
ATTEND_QUANTISED_JOIN(f32, float, 64)
ATTEND_QUANTISED_JOIN(f32, float, 128)
ATTEND_QUANTISED_JOIN(f32, float, 256)

