// Argument blocks of the attention kernels with masks, caps and distance biases (attend_*.h), shared by the device code and
// the host launcher.  Each kernel takes exactly one of these by value.
#pragma once
#include <stdint.h>

// A [b, h, n, d] operand: element strides of the first three, unit stride in d.
struct AttendOperand {
  void* data;
  int64_t sb, sh, sn;
};

// 64 queries' first and last (8 bytes each, causal included), and their Spans (16 bytes)
constexpr uint32_t kSpanRecord = 64 * 8 + 16;

// Queries against keys of the same call.  pos(i) = i + shift is the key position of query i.
//   visible(i, j):  first[i] <= j < last[i]  (absent: 0, nk), causal: j <= pos(i)
//   score(i, j)  =  cap tanh(scale q_i.k_j / cap) - slope |pos(i) - j|
struct AttendParams {
  AttendOperand q, k, v, o;
  AttendOperand grad_o, grad_q, grad_k, grad_v;  // backward
  float* lse;         // [b, hq, nq], natural logarithm
  float* rows;        // backward and key weights: [b, hq, blocks of 64 queries, 64] pairs, see prepare_body
  const int* first;   // [b, nq] or null
  const int* last;    // [b, nq] or null
  const float* slopes;  // [hq] or null
  char* spans;        // ... and, where there is a first or a last, [b, blocks of 64 queries] records of kSpanRecord bytes
  // The work on keys: `shares` workgroups per key head walk equal runs of the (key tile, query head, query tile) triples in which
  // some query sees some key.  A workgroup that did not see all of a key tile leaves its share of the result in a partial buffer:
  int* plan;          // [b, 2 tiles + 1]: first query tile of every key tile, then how many triples of a key head lie before it
  float* partial_k;   // [b, hkv, shares, 2, tile_keys, d]: slot 0 for a tile that it entered in the middle, 1 for one that it left
  float* partial_v;   // (key weights: partial_k [b, hkv, shares, 2, tile_keys])
  const float* weights_in;  // key weights: [b, hkv, nk] or null
  float* weights_out;
  float scale, cap;
  int32_t shift;      // nk - nq
  uint32_t causal;
  uint32_t b, hq, hkv, group, nq, nk, d;
  uint32_t tiles;     // query tiles (forward, grad_q) or key tiles (grad_k / grad_v, key weights) of a head
  uint32_t shares, tile_keys, query_rows;  // ... of a key tile, rows of a query tile
};

// A cache in pages: slot s of a sequence lies in page table[s / page], at slot s % page of it.
struct AttendCache {
  void* k;
  void* v;
  int64_t k_page, k_head, k_slot;  // element strides
  int64_t v_page, v_head, v_slot;
  const int* table;       // [b, table_stride]; null: sequence b is page b
  int64_t table_stride;
  uint32_t page;
  uint32_t pages;         // pages the cache has: an entry of the table past them is taken for page 0
};

struct TreeParams {
  AttendOperand q, o;
  AttendCache cache;
  const int* lengths;      // [b]: slots before the drafted tokens
  const int* start;        // [b] or null (lengths): position of the first drafted token
  const int* positions;    // [b, hkv, positions_stride] or null (the slot itself)
  int64_t positions_stride;
  const uint64_t* visible;  // [b, nodes] (visible_stride 0: [nodes] for all), null: a chain
  int64_t visible_stride;
  const float* slopes;
  float* lse;              // [b, hq, nodes]
  // Units of `unit` keys, a key head after the other, are dealt out to `runs` workgroups (per row tile).  What a workgroup has of a
  // head that others have a share of goes to one of two slots of its own.
  float* partial_o;        // [runs, 2, rows, d] f32, normalised
  float* partial_lse;      // [runs, 2, rows], base 2
  int* head_runs;          // [b, hkv, 2]: first and last run of a head (null: nothing is joined)
  float* head_lse;         // [b, hkv, rows], base 2, of the heads that one run had all of (weights wanted)
  float* scores;           // [b, hkv, counted rows, score_stride], base 2 (weights wanted)
  const float* weights_in;  // [b, hkv, weights_stride]
  float* weights_out;
  int64_t weights_in_stride, weights_out_stride;
  uint64_t counted;        // nodes whose weights are added
  float scale, cap;
  uint32_t b, hq, hkv, group, nodes, d;
  uint32_t max_length;     // no sequence has more slots, drafted tokens included
  uint32_t unit, runs, score_stride;  // (score_stride: max_length in whole units)
  uint32_t whole_heads;    // run n is key head n
  uint32_t page_magic, page_shift;    // key / page = key * page_magic >> page_shift for keys below 2^31
  uint32_t rows, row_tiles;  // group * nodes, and tiles of them
  uint32_t counted_nodes;
};

struct EvictParams {
  AttendCache from, to;
  const int* lengths;
  const float* weights;    // [b, hkv, weights_stride]
  const int* positions;    // [b, hkv, positions_stride] or null (the slot itself)
  int64_t weights_stride, positions_stride;
  float* weights_out;      // [b, hkv, out_stride]
  int* positions_out;      // [b, hkv, out_stride]
  int* chosen;             // [b, hkv, keep]: slots that stay (workspace)
  int* lengths_out;        // [b]
  int64_t out_stride;
  uint32_t b, hkv, d, keep, recent, max_length;
  uint32_t row_bytes;      // d elements in bytes
  uint32_t tiles;          // gather: tiles of kept rows
};
