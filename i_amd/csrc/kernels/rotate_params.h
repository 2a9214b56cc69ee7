// Argument block of the kernels that normalise and turn the heads of queries and keys (rotate.h), shared with the host launcher.
#pragma once
#include <stdint.h>

// A [b, h, n, d] operand: element strides of the first three, unit stride in d.
struct RotateOperand {
  void* data;
  int64_t sb, sh, sn;
};

// queries, or keys
struct RotateSide {
  RotateOperand x, y;  // operand and result (backward: y is the gradient of x)
  RotateOperand g;     // backward: gradient of the result
  const void* weight;  // [d], or null: no norm
  float* partial;      // backward: [workgroups over tokens x chunks, d] shares of the weight's gradient
  void* weight_grad;   // [d]
  uint32_t heads, chunks;  // chunks: runs of p.each heads that a workgroup has
};

struct RotateParams {
  RotateSide side[2];
  const int* positions;  // [axes, b, n]
  int64_t position_axis, position_b;  // element strides, unit stride in n
  const float* frequencies;  // [pairs]
  const int* axis_of;        // [pairs] or null: the first axis
  float eps, inverse_d;
  uint32_t b, n, d, pairs, axes;
  uint32_t tokens;      // b n
  uint32_t each;        // heads of a chunk
  uint32_t steps;       // workgroups over tokens, each of which takes every steps-th tile
  uint32_t tiles;       // tiles of tokens (a wavefront's rows)
  uint32_t f32_weights;  // the weights' type is f32, not the operands'
};
