// Entry points of include/i_rotate.h: checks of arguments, choice of kernels, launches.
#include "../../../include/i_rotate.h"

#include <utility>

#include "../kernels/rotate_params.h"
#include "launch_checks.h"

namespace {

using namespace ihip::host;

// An operand and a result may be the same rows, in the same order.
Err check_in_place(const char* what, const i_attend_tensor* x, const i_attend_tensor* y) {
  if (x->data == y->data && (x->stride_b != y->stride_b || x->stride_h != y->stride_h || x->stride_n != y->stride_n))
    return std::string(what) + " starts where its operand does, with other strides";
  return {};
}

RotateOperand operand(const i_attend_tensor* t) { return RotateOperand{t->data, t->stride_b, t->stride_h, t->stride_n}; }

struct Plan {
  RotateParams p{};
  int lanes = 4;  // of a row
  const char* kind = "";
  bool empty = false;
};

// How the pairs of columns lie, by the kernels' names.  (quads: the lanes of a row hold its pairs, eight each, and its other columns,
// sixteen each)
const char* kind_of(const i_rotate_problem* a, int lanes) {
  if (a->interleaved) return "neighbours";
  if (a->pairs % 8 == 0) return "halves";
  return a->pairs % 4 == 0 && ceil_div(a->pairs, 8) + ceil_div(a->d - 2 * a->pairs, 16) <= lanes ? "quads" : "apart";
}

Err plan_of(const i_rotate_problem* a, bool backward, Plan& plan) {
  if (!a) return "problem is missing";
  if (Err e = check_common(a->dtype, a->b, std::max<int64_t>(a->hq, 1), 1, a->d, 1.0, 0.0); !e.empty()) return e;
  if (a->hq < 0 || a->hkv < 0 || a->hkv > 65535 || a->hq + a->hkv < 1) return "heads must be 0 .. 65535, and one at least";
  if (Err e = check_extent("n", a->n); !e.empty()) return e;
  if (a->b * a->n > kMaxExtent) return "more than 2^30 tokens";
  if (a->pairs < 0 || 2 * a->pairs > a->d) return "pairs must be 0 .. d / 2, not " + std::to_string(a->pairs);
  if (a->interleaved != 0 && a->interleaved != 1) return "interleaved must be 0 or 1";
  if (!std::isfinite(a->eps) || a->eps < 0.0) return "eps must be finite and not negative";
  if ((a->q_weight || a->k_weight) && a->weight_dtype != a->dtype && a->weight_dtype != I_DTYPE_F32) return "the weights' type must be the operands' or f32";
  if ((uintptr_t)a->q_weight % 16 != 0 || (uintptr_t)a->k_weight % 16 != 0) return "a weight must start on a 16-byte boundary";
  if (a->pairs > 0) {
    if (a->axes < 1 || a->axes > 65535) return "axes must be 1 .. 65535";
    if (a->b * a->n > 0 && (!a->positions || !a->frequencies)) return "positions or frequencies: null device pointer";
    if (a->position_stride_axis < 0 || a->position_stride_b < 0) return "negative strides are not supported";
  }
  RotateParams& p = plan.p;
  p.side[0].weight = a->q_weight;
  p.side[1].weight = a->k_weight;
  p.side[0].heads = (uint32_t)a->hq;
  p.side[1].heads = (uint32_t)a->hkv;
  p.positions = a->positions;
  p.position_axis = a->position_stride_axis;
  p.position_b = a->position_stride_b;
  p.frequencies = a->frequencies;
  p.axis_of = a->axis_of;
  p.eps = (float)a->eps;
  p.inverse_d = 1.0f / (float)a->d;
  p.b = (uint32_t)a->b;
  p.n = (uint32_t)a->n;
  p.d = (uint32_t)a->d;
  p.pairs = (uint32_t)a->pairs;
  p.axes = (uint32_t)a->axes;
  p.tokens = (uint32_t)(a->b * a->n);
  p.f32_weights = a->weight_dtype == I_DTYPE_F32;
  plan.empty = p.tokens == 0;
  plan.lanes = a->d <= 64 ? 4 : a->d <= 128 ? 8 : 16;
  plan.kind = kind_of(a, plan.lanes);
  p.tiles = (uint32_t)ceil_div(p.tokens, 64 / plan.lanes);
  // Heads of a workgroup: 16, four for each wavefront, whose angles then cost little, or fewer where that leaves the chip less than 2048
  // workgroups (a multiple of four).  4 x 4096 tokens of 32 and 8 heads of 128 columns, bf16, us with 4, 8, 16, 32 heads: 110, 76, 66,
  // 77, backward too 229, 165, 144, 169;  with 2048, 4096, 8192 workgroups at least: 6001 tokens of 16 and 16 heads of 72 16.4, 18.5, 25.4, 4096 of
  // 32 and 8 of 128 21.3, 17.6, 22.8.
  const int64_t heads = a->hq + a->hkv, fours = ceil_div(heads, 4), runs = std::max<int64_t>(ceil_div(heads, 16), std::min(fours, 2048 / std::max<int64_t>(1, p.tiles)));
  p.each = (uint32_t)(4 * ceil_div(fours, runs));
  for (RotateSide& side : p.side) side.chunks = (uint32_t)ceil_div(side.heads, p.each);
  const int64_t chunks = p.side[0].chunks + p.side[1].chunks;
  p.steps = (uint32_t)std::min<int64_t>(p.tiles, kMaxThreads / 256 / chunks);
  if (backward && (a->q_weight || a->k_weight)) {
    // Each of them leaves a share of the weights' gradients: as many as the chip holds at once.  (Dealt out evenly, which is fewer: 4096
    // tokens of 16 and 16 heads of 256 columns 30 -> 32 us.)
    const int64_t held = a->dtype == I_DTYPE_BF16 && plan.kind[0] != 'a' ? 3 : 2;
    p.steps = (uint32_t)std::min<int64_t>(p.tiles, std::max<int64_t>(1, 256 * held / chunks));
  }
  return {};
}

std::string kernel_name(const char* kernel, const i_rotate_problem* a, const Plan& plan) {
  return std::string(kernel) + type_name(a->dtype) + "_" + plan.kind + "_l" + std::to_string(plan.lanes);
}

Err run_rows(const char* kernel, const i_rotate_problem* a, const Plan& plan, hipStream_t stream) {
  const RotateParams& p = plan.p;
  return run(kernel_name(kernel, a, plan), ihip::CodeObject::Rotate, (int64_t)p.steps * (p.side[0].chunks + p.side[1].chunks), 256, p, stream);
}

Err forward(const i_rotate_problem* a, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* q_out,
            const i_attend_tensor* k_out, hipStream_t stream) {
  Plan plan;
  if (Err e = plan_of(a, false, plan); !e.empty()) return e;
  if (plan.empty) return {};
  const std::pair<const i_attend_tensor*, const i_attend_tensor*> given[2] = {{q, q_out}, {k, k_out}};
  for (int n = 0; n < 2; ++n) {
    RotateSide& side = plan.p.side[n];
    if (side.heads == 0) continue;
    if (Err e = check_tensor(n ? "k" : "q", given[n].first, a->dtype); !e.empty()) return e;
    if (Err e = check_tensor(n ? "k_out" : "q_out", given[n].second, a->dtype); !e.empty()) return e;
    if (Err e = check_in_place(n ? "k_out" : "q_out", given[n].first, given[n].second); !e.empty()) return e;
    side.x = operand(given[n].first);
    side.y = operand(given[n].second);
  }
  return run_rows("rotate_", a, plan, stream);
}

// The shares of the weights' gradients in the workspace; returns its bytes.
size_t carve(Plan& plan, char* base) {
  Carver c{base};
  for (RotateSide& side : plan.p.side)
    if (side.weight && side.heads > 0) side.partial = c.take<float>((int64_t)plan.p.steps * side.chunks * plan.p.d);
  return c.at;
}

Err backward(const i_rotate_problem* a, const i_attend_tensor* go_q, const i_attend_tensor* go_k, const i_attend_tensor* q, const i_attend_tensor* k,
             const i_attend_tensor* gq, const i_attend_tensor* gk, void* gq_weight, void* gk_weight, void* workspace, size_t workspace_bytes,
             hipStream_t stream) {
  Plan plan;
  if (Err e = plan_of(a, true, plan); !e.empty()) return e;
  struct {
    const i_attend_tensor *go, *x, *gx;
    void* weight;
  } const given[2] = {{go_q, q, gq, gq_weight}, {go_k, k, gk, gk_weight}};
  bool join = false;
  for (int n = 0; n < 2; ++n) {
    RotateSide& side = plan.p.side[n];
    if (side.weight) {
      if (!given[n].weight) return "the gradient of a weight: null device pointer";
      side.weight_grad = given[n].weight;
      join = true;
    }
    if (plan.empty || side.heads == 0) continue;
    if (Err e = check_tensor(n ? "grad_k_out" : "grad_q_out", given[n].go, a->dtype); !e.empty()) return e;
    if (Err e = check_tensor(n ? "grad_k" : "grad_q", given[n].gx, a->dtype); !e.empty()) return e;
    if (Err e = check_in_place(n ? "grad_k" : "grad_q", given[n].go, given[n].gx); !e.empty()) return e;
    side.g = operand(given[n].go);
    side.y = operand(given[n].gx);
    if (!side.weight) continue;
    if (Err e = check_tensor(n ? "k" : "q", given[n].x, a->dtype); !e.empty()) return e;
    side.x = operand(given[n].x);
  }
  if (Err e = check_workspace(workspace, workspace_bytes, carve(plan, (char*)workspace)); !e.empty()) return e;
  if (!plan.empty)
    if (Err e = run_rows("rotate_grad_", a, plan, stream); !e.empty()) return e;
  if (!join) return {};
  // (without a row the sum is of no shares: zeros)
  return run(std::string("rotate_join_") + type_name(a->dtype), ihip::CodeObject::Rotate, ceil_div(a->d, 32), 1024, plan.p, stream, 2);
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

int i_rotate(const i_rotate_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* q_out,
             const i_attend_tensor* k_out, void* stream) {
  return guarded("rotate", [&] { return forward(problem, q, k, q_out, k_out, (hipStream_t)stream); });
}

size_t i_rotate_backward_workspace(const i_rotate_problem* problem) {
  size_t bytes = (size_t)-1;
  guarded("rotate_backward", [&] {
    Plan plan;
    if (Err e = plan_of(problem, true, plan); !e.empty()) return e;
    bytes = carve(plan, nullptr);
    return Err{};
  });
  return bytes;
}

int i_rotate_backward(const i_rotate_problem* problem, const i_attend_tensor* grad_q_out, const i_attend_tensor* grad_k_out,
                      const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* grad_q, const i_attend_tensor* grad_k,
                      void* grad_q_weight, void* grad_k_weight, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("rotate_backward", [&] {
    return backward(problem, grad_q_out, grad_k_out, q, k, grad_q, grad_k, grad_q_weight, grad_k_weight, workspace, workspace_bytes, (hipStream_t)stream);
  });
}

}  // extern "C"
#pragma GCC visibility pop
