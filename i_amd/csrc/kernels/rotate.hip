// The code object of the norm and rotary position of queries and keys.
#include "rotate.h"

#define ROTATE(TYPE, T, LPR, NAME, KIND)                                                                                  \
  extern "C" __global__ void __launch_bounds__(256) rotate_##TYPE##_##NAME##_l##LPR(RotateParams p) {                     \
    rotate::forward_body<T, LPR, rotate::KIND>(p);                                                                        \
  }                                                                                                                       \
  extern "C" __global__ void __launch_bounds__(256) rotate_grad_##TYPE##_##NAME##_l##LPR(RotateParams p) {                \
    rotate::backward_body<T, LPR, rotate::KIND>(p);                                                                       \
  }
#define ROTATES(TYPE, T, LPR) \
  ROTATE(TYPE, T, LPR, halves, kHalves) ROTATE(TYPE, T, LPR, quads, kQuads) ROTATE(TYPE, T, LPR, neighbours, kNeighbours) ROTATE(TYPE, T, LPR, apart, kApart)
ROTATES(bf16, bf16_t, 4)
ROTATES(bf16, bf16_t, 8)
ROTATES(bf16, bf16_t, 16)
ROTATES(f32, float, 4)
ROTATES(f32, float, 8)
ROTATES(f32, float, 16)

extern "C" __global__ void __launch_bounds__(1024) rotate_join_bf16(RotateParams p) { rotate::join_body<bf16_t>(p); }
extern "C" __global__ void __launch_bounds__(1024) rotate_join_f32(RotateParams p) { rotate::join_body<float>(p); }
