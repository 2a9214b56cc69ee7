// The code object of the norm and rotary position of queries and keys.
#include "rotate.h"

// (OCC: workgroups that a compute unit holds, which the launcher counts on)
#define ROTATE(TYPE, T, LPR, NAME, KIND, OCC)                                                                             \
  extern "C" __global__ void __launch_bounds__(256) rotate_##TYPE##_##NAME##_l##LPR(RotateParams p) {                     \
    rotate::forward_body<T, LPR, rotate::KIND>(p);                                                                        \
  }                                                                                                                       \
  extern "C" __global__ void __launch_bounds__(256, OCC) rotate_grad_##TYPE##_##NAME##_l##LPR(RotateParams p) {           \
    rotate::backward_body<T, LPR, rotate::KIND>(p);                                                                       \
  }
#define ROTATES(TYPE, T, LPR, OCC)                                                                                        \
  ROTATE(TYPE, T, LPR, halves, kHalves, OCC) ROTATE(TYPE, T, LPR, quads, kQuads, OCC)                                     \
  ROTATE(TYPE, T, LPR, neighbours, kNeighbours, OCC) ROTATE(TYPE, T, LPR, apart, kApart, 2)
ROTATES(bf16, bf16_t, 4, 3)
ROTATES(bf16, bf16_t, 8, 3)
ROTATES(bf16, bf16_t, 16, 3)
ROTATES(f32, float, 4, 2)
ROTATES(f32, float, 8, 2)
ROTATES(f32, float, 16, 2)

extern "C" __global__ void __launch_bounds__(1024) rotate_join_bf16(RotateParams p) { rotate::join_body<bf16_t>(p); }
extern "C" __global__ void __launch_bounds__(1024) rotate_join_f32(RotateParams p) { rotate::join_body<float>(p); }
