// The code object of the attention kernels with masks: forward.
#include "attend_forward.h"

#define ATTEND_FORWARD(TYPE, T, DPAD, DUSE, BN, NW, QB, OCC)                                                              \
  extern "C" __global__ void __launch_bounds__(64 * NW, OCC) attend_fwd_##TYPE##_d##DUSE(AttendParams p) {                 \
    attend::forward_body<T, DPAD, DUSE, BN, NW, QB>(p);                                                                   \
  }
ATTEND_FORWARD(bf16, bf16_t, 64, 64, 64, 4, 2, 2)
ATTEND_FORWARD(bf16, bf16_t, 128, 96, 64, 4, 2, 2)
ATTEND_FORWARD(bf16, bf16_t, 128, 128, 64, 4, 2, 2)
ATTEND_FORWARD(bf16, bf16_t, 256, 256, 64, 4, 2, 1)
ATTEND_FORWARD(f32, float, 64, 64, 32, 4, 2, 3)
ATTEND_FORWARD(f32, float, 128, 96, 32, 4, 2, 2)
ATTEND_FORWARD(f32, float, 128, 128, 32, 4, 2, 2)
ATTEND_FORWARD(f32, float, 256, 256, 32, 4, 1, 1)

#define ATTEND_HALVES(TYPE, T, DPAD, DUSE)                                                                                 \
  extern "C" __global__ void __launch_bounds__(512, 2) attend_fwd_halves_##TYPE##_d##DUSE(AttendParams p) {                \
    attend::forward_body<T, DPAD, DUSE, 64, 8, 1, 2>(p);                                                                  \
  }
ATTEND_HALVES(bf16, bf16_t, 64, 64)
ATTEND_HALVES(bf16, bf16_t, 128, 96)
ATTEND_HALVES(bf16, bf16_t, 128, 128)
ATTEND_HALVES(bf16, bf16_t, 256, 256)
ATTEND_HALVES(f32, float, 64, 64)
ATTEND_HALVES(f32, float, 128, 96)
ATTEND_HALVES(f32, float, 128, 128)

#define ATTEND_FEW(TYPE, T, DPAD, DUSE, NW)                                                                       \
  extern "C" __global__ void __launch_bounds__(64 * NW, 1) attend_fwd_few_##TYPE##_d##DUSE(AttendParams p) {       \
    attend::forward_few_body<T, DPAD, DUSE, NW>(p);                                                               \
  }
ATTEND_FEW(bf16, bf16_t, 64, 64, 8)
ATTEND_FEW(bf16, bf16_t, 128, 128, 4)
ATTEND_FEW(bf16, bf16_t, 256, 256, 2)
ATTEND_FEW(f32, float, 64, 64, 4)
ATTEND_FEW(f32, float, 128, 128, 2)
ATTEND_FEW(f32, float, 256, 256, 1)
