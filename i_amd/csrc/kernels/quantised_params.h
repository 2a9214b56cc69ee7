// Argument blocks of the kernels of a cache in 8 or 4 bits (quantised.h, attend_quantised.h), shared with the host launcher.
#pragma once
#include "attend_params.h"

// The keys, or the values: strides in bytes.
struct QuantisedSide {
  uint8_t* codes;
  uint8_t* scales;
  int64_t page, head, slot;
  int64_t scale_page, scale_head, scale_slot;
};

struct QuantisedTreeParams {
  TreeParams tree;  // (its cache: pages and table alone)
  QuantisedSide k, v;
};

// A launch has at most 2^32 threads along x: workgroups 2^kMoveAcross y + x.
constexpr uint32_t kMoveAcross = 23;

// Tokens to or from a cache: token t of sequence b is slot first[b] + t, for t < counts[b].
struct QuantisedMoveParams {
  AttendOperand k, v;  // [b, hkv, n, d]
  QuantisedSide k_cache, v_cache;
  const int* table;    // as AttendCache
  int64_t table_stride;
  const int* first;    // [b] or null: 0
  const int* counts;   // [b] or null: n
  uint32_t page, pages, page_magic, page_shift;
  uint32_t slots;      // of a sequence: what its pages hold
  uint32_t b, hkv, n, d;
  uint32_t rows;       // b hkv n
  uint32_t head_magic, head_shift, token_magic, token_shift;  // divisions by hkv and n
};
