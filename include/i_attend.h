/*
 * Attention with masks, capped scores and a bias by distance, its gradient, and attention over a cache: hand-written
 * gfx950 kernels beside those of i_hip.h.  The reference has none of them (its attention component has no mask and no
 * gradient: ilang-python/flash-attn.py:45-55).
 *
 * All `void*`, `int*` and `float*` operands are device pointers; `stream` is a hipStream_t (NULL = the default stream).
 * Launches are asynchronous on that stream, allocate nothing and keep nothing from call to call.  Return value 0 =
 * enqueued, -1 = refused with the text in i_error(); nothing is enqueued by a call that is refused.
 *
 *   score(i, j) = cap tanh(scale q_i.k_j / cap) - slope_h |pos(i) - j|       (cap 0: no cap; no slopes: no bias)
 *   p(i, j)     = exp(score(i, j) - lse(i)) over the keys that query i sees,   o(i) = sum_j p(i, j) v_j
 *
 * A query that sees no key gives o = 0, lse = -inf and no gradient, whatever its q and grad_o hold.  Keys that no query of a
 * call sees may hold anything, NaN included, between keys that are seen too; so may a drafted token's slot that no node
 * sees.  A key that some query sees and others do not must be finite in v for those others (its weight 0 is multiplied
 * with it).  Sums, maxima, lse and gradients' sums are f32; with bf16 operands the probabilities are rounded to bf16
 * before the second product, as its other operand is, and the gradient's score gradients to two bf16 parts.
 * Exponentials are divided by their sum at the end: those of a tile may add up to 2^32 before their reference follows, those of 2^30 keys
 * to 2^57, so that magnitudes in v above 2^70 may give infinities or NaN where the result would be finite.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "i_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A [b, h, n, d] tensor: strides in elements, unit stride in d.  The address and every stride are multiples of 16 bytes. */
typedef struct {
  void* data;
  int64_t stride_b, stride_h, stride_n;
} i_attend_tensor;

/* hq is a multiple of hkv: query heads h (hq / hkv) .. share key head h.  d: a multiple of 8 up to 256. */
typedef struct {
  int64_t dtype; /* I_DTYPE_*, of q, k, v, o and their gradients */
  int64_t b, hq, hkv, nq, nk, d;
  double scale;
  double cap;          /* 0: scores as they are */
  const float* slopes; /* [hq] or NULL */
  int64_t causal;      /* 1: query i sees j <= pos(i) = i + nk - nq */
  const int* first;    /* [b, nq] or NULL: query i sees j >= first[i] */
  const int* last;     /* [b, nq] or NULL: query i sees j < last[i] */
} i_attend_problem;

/* o and lse ([b, hq, nq] f32, natural logarithm; may be NULL). */
int i_attend(const i_attend_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const i_attend_tensor* v,
             const i_attend_tensor* o, float* lse, void* stream);

/*
 * Bytes of device memory (256-byte aligned) that the call below works in; (size_t)-1 + i_error for a bad problem.  The work on
 * keys is counted in tiles of 64 or 128 keys and 32 or 64 queries of a query head: 2^31 of them for a key head are refused.
 */
size_t i_attend_backward_workspace(const i_attend_problem* problem);

/* grad_q, grad_k, grad_v from grad_o and what the forward call took and gave.  Sums are added in a fixed order. */
int i_attend_backward(const i_attend_problem* problem, const i_attend_tensor* grad_o, const i_attend_tensor* q,
                      const i_attend_tensor* k, const i_attend_tensor* v, const i_attend_tensor* o, const float* lse,
                      const i_attend_tensor* grad_q, const i_attend_tensor* grad_k, const i_attend_tensor* grad_v,
                      void* workspace, size_t workspace_bytes, void* stream);

size_t i_attend_weights_workspace(const i_attend_problem* problem);

/*
 * What every key received: weights_out[b, hkv, j] = weights_in[b, hkv, j] + sum over its query heads and queries of p(i, j).
 * weights_in (dense, like weights_out) may be NULL (zeros) or weights_out itself.
 */
int i_attend_weights(const i_attend_problem* problem, const i_attend_tensor* q, const i_attend_tensor* k, const float* lse,
                     const float* weights_in, float* weights_out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * A cache in pages: slot s of sequence b is slot s % page of page table[b, s / page].  k and v: [pages, hkv, page, d] with
 * strides in elements as above.  table NULL: sequence b is page b.  An entry outside 0 .. pages - 1 reads as page 0
 * and is not written.
 */
typedef struct {
  void *k, *v;
  int64_t k_stride_page, k_stride_head, k_stride_slot;
  int64_t v_stride_page, v_stride_head, v_stride_slot;
  const int* table;
  int64_t table_stride; /* entries of a sequence */
  int64_t page, pages;
} i_attend_cache;

/*
 * `nodes` (1 .. 64) drafted tokens of every sequence against its cache: q [b, hq, nodes, d].  Slots 0 .. lengths[b] - 1 are
 * seen by every node, slot lengths[b] + u (where the keys of node u already lie) by the nodes t with bit u of
 * visible[b, t] set.  pos(t) = start[b] + number of bits of visible[b, t] - 1; a slot below lengths[b] is at
 * positions[b, hkv, slot], or at its own index.  One node that sees itself is the step of a single token.
 */
typedef struct {
  int64_t dtype;
  int64_t b, hq, hkv, nodes, d;
  double scale, cap;
  const float* slopes;
  const int* lengths;      /* [b] */
  int64_t max_length;      /* no lengths[b] + nodes is larger (a larger one is cut) */
  const int* start;        /* [b] or NULL: lengths */
  const int* positions;    /* [b, hkv, positions_stride] or NULL */
  int64_t positions_stride;
  const int64_t* visible;  /* [b, nodes], or [nodes] with visible_stride 0; NULL: a chain, node t sees 0 .. t */
  int64_t visible_stride;
  const float* weights_in; /* [b, hkv, stride] or NULL; with weights_out: out = in + p of the counted nodes, max_length entries */
  float* weights_out;      /* may be weights_in itself */
  int64_t weights_in_stride, weights_out_stride;
  int64_t counted;         /* bit t: the weights of node t count */
} i_attend_tree_problem;

size_t i_attend_tree_workspace(const i_attend_tree_problem* problem);
int i_attend_tree(const i_attend_tree_problem* problem, const i_attend_tensor* q, const i_attend_cache* cache,
                  const i_attend_tensor* o, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Cuts every sequence's cache to `keep` entries a key head: the last `recent` slots stay, and of those before them the
 * keep - recent of largest weight (of equal ones the lowest slots; NaN counts as the smallest).  They move to the cache `to`
 * in the order of their slots, slot 0 on; a sequence of at most `keep` entries moves whole.  weights_out, positions_out
 * ([b, hkv, out_stride]) get the weights and positions (the slot where `positions` is NULL) of what stays, lengths_out the
 * new lengths.  Nothing is written past them.  The pages of `to` must not be pages of `from`, and
 * the new lengths, weights and positions that share memory with the old ones are refused.
 */
typedef struct {
  int64_t dtype;
  int64_t b, hkv, d, keep, recent, max_length;
  const int* lengths;
  const float* weights; /* [b, hkv, weights_stride] */
  int64_t weights_stride;
  const int* positions; /* [b, hkv, positions_stride] or NULL */
  int64_t positions_stride;
  float* weights_out;
  int* positions_out;
  int64_t out_stride;
  int* lengths_out; /* [b] */
} i_evict_problem;

size_t i_evict_workspace(const i_evict_problem* problem);
int i_evict(const i_evict_problem* problem, const i_attend_cache* from, const i_attend_cache* to, void* workspace,
            size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
