// What the launchers of trees of drafted tokens share, whatever their cache holds.
#pragma once
#include "../kernels/attend_params.h"
#include "launch_checks.h"

namespace ihip::host {

inline AttendOperand operand(const i_attend_tensor* t) { return t ? AttendOperand{t->data, t->stride_b, t->stride_h, t->stride_n} : AttendOperand{}; }

// n / divisor as a product and a shift for n below 2^31: with 2^l >= divisor > 2^(l - 1) and the product by 2^(31 + l) / divisor rounded
// up, off by less than n 2^l / 2^(31 + l) < 1 / divisor
struct Divider {
  uint32_t magic, shift;
  explicit Divider(uint32_t divisor) {
    int l = 0;
    while ((1ll << l) < divisor) ++l;
    magic = (uint32_t)(((1ull << (31 + l)) + divisor - 1) / divisor);
    shift = (uint32_t)(31 + l);
  }
};

// Checks the problem's sizes and fills in what follows from it alone.
inline Err tree_problem(const i_attend_tree_problem* a, TreeParams& p) {
  if (!a) return "problem is missing";
  if (Err e = check_common(a->dtype, a->b, a->hq, a->hkv, a->d, a->scale, a->cap); !e.empty()) return e;
  if (a->nodes < 1 || a->nodes > 64) return "nodes must be 1 .. 64, not " + std::to_string(a->nodes);
  if (a->max_length < a->nodes || a->max_length > kMaxExtent) return "max_length must be at least the number of nodes and at most 2^30";
  if (a->visible_stride < 0 || a->positions_stride < 0 || a->weights_in_stride < 0 || a->weights_out_stride < 0) return "negative strides are not supported";
  p.lengths = a->lengths;
  p.start = a->start;
  p.positions = a->positions;
  p.positions_stride = a->positions_stride;
  p.visible = (const uint64_t*)a->visible;
  p.visible_stride = a->visible_stride;
  p.slopes = a->slopes;
  p.weights_in = a->weights_in;
  p.weights_out = a->weights_out;
  p.weights_in_stride = a->weights_in_stride;
  p.weights_out_stride = a->weights_out_stride;
  p.counted = (uint64_t)a->counted & (a->nodes == 64 ? ~0ull : (1ull << a->nodes) - 1);
  p.scale = (float)a->scale;
  p.cap = (float)a->cap;
  p.b = (uint32_t)a->b;
  p.hq = (uint32_t)a->hq;
  p.hkv = (uint32_t)a->hkv;
  p.group = (uint32_t)(a->hq / a->hkv);
  p.nodes = (uint32_t)a->nodes;
  p.d = (uint32_t)a->d;
  p.max_length = (uint32_t)a->max_length;
  p.rows = p.group * p.nodes;
  p.counted_nodes = (uint32_t)__builtin_popcountll(p.counted);
  return {};
}

// the device arrays of a problem that has sequences
inline Err check_tree_arrays(const i_attend_tree_problem* a) {
  if (!a->lengths) return "lengths: null device pointer";
  if ((a->weights_in != nullptr) != (a->weights_out != nullptr)) return "weights_in and weights_out go together";
  if (a->weights_out && (a->weights_in_stride < a->max_length || a->weights_out_stride < a->max_length)) return "weights must have max_length entries a head";
  if (a->positions && a->positions_stride < a->max_length - a->nodes) return "positions must have an entry for every slot before the drafted tokens";
  if (a->visible && a->visible_stride != 0 && a->visible_stride < a->nodes) return "visible must have an entry for every node";
  return {};
}

}  // namespace ihip::host
