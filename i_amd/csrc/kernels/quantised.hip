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

#define ATTEND_QUANTISED_ROWS(TYPE, T, BITS, DPAD, BN, RT, OCC)                                                                           \
  extern "C" __global__ void __launch_bounds__(256, OCC) attend_quantised_##TYPE##_b##BITS##_d##DPAD##_rows(QuantisedTreeParams p) { \
    attend::quantised_rows_body<T, BITS, DPAD, BN, RT>(p);                                                                           \
  }
#define ATTEND_QUANTISED(BITS)                                \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 64, 64, 2, 2)     \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 128, 32, 2, 2)    \
  ATTEND_QUANTISED_ROWS(bf16, bf16_t, BITS, 256, 32, 1, 2)    \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 64, 32, 2, 2)       \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 128, 32, 1, 2)      \
  ATTEND_QUANTISED_ROWS(f32, float, BITS, 256, 32, 1, 1)
ATTEND_QUANTISED(4)
ATTEND_QUANTISED(8)
