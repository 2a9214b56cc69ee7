// The code object of the attention kernels with masks: gradients and the weights of keys.
#include "attend_backward.h"

#define ATTEND_PREPARE(TYPE, T)                                                                         \
  extern "C" __global__ void __launch_bounds__(256, 5) attend_prepare_##TYPE(AttendParams p) {          \
    attend::prepare_body<T, true>(p);                                                                   \
  }                                                                                                     \
  extern "C" __global__ void __launch_bounds__(256) attend_join_gradients_##TYPE(AttendParams p) {      \
    attend::join_gradients_body<T>(p);                                                                  \
  }
ATTEND_PREPARE(bf16, bf16_t)
ATTEND_PREPARE(f32, float)
extern "C" __global__ void __launch_bounds__(256) attend_prepare_weights(AttendParams p) { attend::prepare_body<float, false>(p); }
extern "C" __global__ void __launch_bounds__(256) attend_join_weights(AttendParams p) { attend::join_weights_body(p); }

#define ATTEND_BACKWARD(TYPE, T, DPAD, DUSE, BQ, NW, KB, OCC, BN, QB, QOCC)                                         \
  extern "C" __global__ void __launch_bounds__(64 * NW, OCC) attend_grad_keys_##TYPE##_d##DUSE(AttendParams p) {    \
    attend::keys_body<T, DPAD, DUSE, BQ, NW, KB, true>(p);                                                          \
  }                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(64 * NW, QOCC) attend_grad_queries_##TYPE##_d##DUSE(AttendParams p) { \
    attend::queries_body<T, DPAD, DUSE, BN, NW, QB>(p);                                                             \
  }
ATTEND_BACKWARD(bf16, bf16_t, 64, 64, 64, 4, 2, 2, 64, 2, 2)
ATTEND_BACKWARD(bf16, bf16_t, 128, 96, 64, 4, 2, 1, 64, 2, 2)
ATTEND_BACKWARD(bf16, bf16_t, 128, 128, 64, 4, 2, 1, 64, 2, 2)
ATTEND_BACKWARD(bf16, bf16_t, 256, 256, 32, 4, 1, 1, 32, 1, 1)
ATTEND_BACKWARD(f32, float, 64, 64, 32, 4, 2, 1, 32, 2, 1)
ATTEND_BACKWARD(f32, float, 128, 96, 32, 4, 1, 1, 32, 2, 1)
ATTEND_BACKWARD(f32, float, 128, 128, 32, 4, 1, 1, 32, 1, 1)
ATTEND_BACKWARD(f32, float, 256, 256, 32, 4, 1, 1, 32, 1, 1)

#define ATTEND_WEIGHTS(TYPE, T, DPAD, DUSE, BQ, NW, KB, OCC)                                                  \
  extern "C" __global__ void __launch_bounds__(64 * NW, OCC) attend_weights_##TYPE##_d##DUSE(AttendParams p) { \
    attend::keys_body<T, DPAD, DUSE, BQ, NW, KB, false>(p);                                                   \
  }
ATTEND_WEIGHTS(bf16, bf16_t, 64, 64, 64, 4, 2, 3)
ATTEND_WEIGHTS(bf16, bf16_t, 128, 96, 64, 4, 2, 3)
ATTEND_WEIGHTS(bf16, bf16_t, 128, 128, 64, 4, 2, 3)
ATTEND_WEIGHTS(bf16, bf16_t, 256, 256, 32, 4, 2, 2)
ATTEND_WEIGHTS(f32, float, 64, 64, 32, 4, 2, 3)
ATTEND_WEIGHTS(f32, float, 128, 96, 32, 4, 2, 2)
ATTEND_WEIGHTS(f32, float, 128, 128, 32, 4, 2, 2)
ATTEND_WEIGHTS(f32, float, 256, 256, 32, 4, 1, 1)

#define ATTEND_QUERIES_HALVES(TYPE, T, DPAD, DUSE)                                                                         \
  extern "C" __global__ void __launch_bounds__(512, 2) attend_grad_queries_halves_##TYPE##_d##DUSE(AttendParams p) {       \
    attend::queries_body<T, DPAD, DUSE, 64, 8, 1, 2>(p);                                                                  \
  }
ATTEND_QUERIES_HALVES(bf16, bf16_t, 64, 64)
ATTEND_QUERIES_HALVES(bf16, bf16_t, 128, 96)
ATTEND_QUERIES_HALVES(bf16, bf16_t, 128, 128)
ATTEND_QUERIES_HALVES(bf16, bf16_t, 256, 256)
ATTEND_QUERIES_HALVES(f32, float, 64, 64)
ATTEND_QUERIES_HALVES(f32, float, 128, 96)
ATTEND_QUERIES_HALVES(f32, float, 128, 128)

#define ATTEND_QUERIES_FEW(TYPE, T, DPAD, DUSE, NW)                                                                       \
  extern "C" __global__ void __launch_bounds__(64 * NW, 1) attend_grad_queries_few_##TYPE##_d##DUSE(AttendParams p) {      \
    attend::queries_few_body<T, DPAD, DUSE, NW>(p);                                                                       \
  }
ATTEND_QUERIES_FEW(bf16, bf16_t, 64, 64, 8)
ATTEND_QUERIES_FEW(bf16, bf16_t, 128, 128, 4)
ATTEND_QUERIES_FEW(bf16, bf16_t, 256, 256, 2)
ATTEND_QUERIES_FEW(f32, float, 64, 64, 4)
ATTEND_QUERIES_FEW(f32, float, 128, 128, 2)
ATTEND_QUERIES_FEW(f32, float, 256, 256, 1)
