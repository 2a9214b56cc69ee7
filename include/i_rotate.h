/*
 * Norm and rotary position of the heads of queries and keys in one pass, and its gradient: what lies between a model's projections and
 * the attention of i_attend.h.  The reference has no counterpart (ilang-python/flash-attn.py:45-55 starts from finished heads).
 *
 *   n = x / sqrt(mean(x^2) + eps),  u = n weight    (per row of d columns; weight NULL: u = x)
 *   y_a = u_a cos t - u_b sin t,  y_b = u_b cos t + u_a sin t,  t = position of the token on the pair's axis * frequency of the pair
 *
 * for `pairs` pairs (a, b) of columns: (j, j + pairs), or with `interleaved` (2 j, 2 j + 1).  The columns from 2 pairs on do not turn.
 * Angles are reduced in 64 bits, sums and rotations are in f32, results are rounded once.
 *
 * Pointers are device pointers, `stream` is a hipStream_t.  Calls allocate nothing and keep nothing; 0 = enqueued, -1 = refused with
 * the text in i_error().
 */
#pragma once

#include "i_attend.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  int64_t dtype;                /* I_DTYPE_* of the operands and results */
  int64_t b, hq, hkv, n, d;     /* hkv 0: no keys.  d: a multiple of 8 up to 256 */
  int64_t pairs;                /* 0 .. d / 2; 0: nothing turns */
  int64_t axes;                 /* axes that a token has positions on */
  int64_t interleaved;
  const int* positions;         /* [axes, b, n]: strides in elements, unit stride in n */
  int64_t position_stride_axis, position_stride_b;
  const float* frequencies;     /* [pairs], radians per position */
  const int* axis_of;           /* [pairs]: the axis of a pair (0 .. axes - 1; others count as the nearest), or NULL: axis 0 */
  const void *q_weight, *k_weight; /* [d] on a 16-byte boundary, or NULL: no norm */
  int64_t weight_dtype;
  double eps;
} i_rotate_problem;

/* q_out and k_out may be q and k themselves (the same address and strides); k and k_out are not looked at where hkv is 0. */
int i_rotate(const i_rotate_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* q_out,
             const i_attend_tensor* k_out, void* stream);

/* Bytes of device memory (256-byte aligned) that the call below works in; (size_t)-1 + i_error for a bad problem. */
size_t i_rotate_backward_workspace(const i_rotate_problem* problem);

/*
 * Gradients of q and k (which may be written over those of the results) and, where there is a norm, of its weight: [d] of
 * weight_dtype, sums over all rows in a fixed order.  Without a norm q, respectively k, is not looked at.
 */
int i_rotate_backward(const i_rotate_problem* problem, const i_attend_tensor* grad_q_out, const i_attend_tensor* grad_k_out,
                      const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* grad_q, const i_attend_tensor* grad_k,
                      void* grad_q_weight, void* grad_k_weight, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
