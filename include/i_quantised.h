/*
 * A cache of keys and values in 8 or 4 bits: tokens written to it, read back, and attention over it (as i_attend_tree over a cache of
 * the operands' own type).  The reference has no counterpart (ilang-python/flash-attn.py:45-55).
 *
 * A row (slot and key head) of d columns, padded with zeros to a multiple of 32, is kept as blocks of 32 columns: a scale 2^(byte - 127)
 * and 32 codes.  bits 4: codes 0 .. 7 are 0, 1/2, 1, 3/2, 2, 3, 4, 6, codes 8 .. 15 their negatives, column 2 j in the low half of
 * byte j.  bits 8: sign, 4 bits of exponent (bias 7), 3 of fraction, the largest 448 (code 127 is NaN).  The scale is the smallest power
 * of two s with max |x| <= 7 s (4 bits), 464 s (8 bits), at least 2^-125 and 2^-117; a code is the number nearest to x / s, of two
 * equally near ones the even code.  A block that holds a NaN, an infinity or a magnitude above 1.75 2^127 has scale byte 255: all of it
 * reads as NaN.  (Smaller scales than those two are never written; blocks of them, but for zeros, may read as anything finite.)
 *
 * Pointers are device pointers, `stream` is a hipStream_t.  Calls allocate nothing and keep nothing; 0 = enqueued, -1 = refused with the
 * text in i_error().
 */
#pragma once

#include "i_attend.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Codes [pages, hkv, page, columns bits / 8] and scales [pages, hkv, page, columns / 32], columns being d rounded up to a multiple of
 * 32: strides in bytes, unit stride in a row; codes start and lie on multiples of 16 bytes.  Pages and table as in i_attend_cache: slot
 * s of sequence b is slot s % page of page table[b, s / page]; an entry outside 0 .. pages - 1 reads as page 0 and is not written.
 */
typedef struct {
  void *k, *k_scales, *v, *v_scales;
  int64_t bits; /* 4 | 8 */
  int64_t k_stride_page, k_stride_head, k_stride_slot;
  int64_t k_scales_stride_page, k_scales_stride_head, k_scales_stride_slot;
  int64_t v_stride_page, v_stride_head, v_stride_slot;
  int64_t v_scales_stride_page, v_scales_stride_head, v_scales_stride_slot;
  const int* table;
  int64_t table_stride; /* entries from the first of a sequence to that of the next */
  int64_t page, pages;
  int64_t listed;       /* entries of a sequence: it has no other pages; 0: table_stride */
} i_quantised_cache;

/* Token t < counts[b] of sequence b is slot first[b] + t. */
typedef struct {
  int64_t dtype; /* I_DTYPE_* of the operands */
  int64_t b, hkv, n, d;
  const int* first;  /* [b] or NULL: 0 */
  const int* counts; /* [b] or NULL: n */
} i_quantised_problem;

/* k, v [b, hkv, n, d] to the cache.  A slot that the sequence's pages do not have is not written. */
int i_quantised_store(const i_quantised_problem* problem, const i_attend_tensor* k, const i_attend_tensor* v, const i_quantised_cache* cache,
                      void* stream);

/* The cache to k, v [b, hkv, n, d].  Tokens past counts[b], and slots that the sequence's pages do not have, are zeros. */
int i_quantised_load(const i_quantised_problem* problem, const i_quantised_cache* cache, const i_attend_tensor* k, const i_attend_tensor* v,
                     void* stream);

/*
 * i_attend_tree over such a cache: the same problem but for the weights, which have to be NULL here.  q and o have the problem's type.
 * Values: what i_attend.h says of large ones holds here, up to 2^70 all are right.  With at most 16 rows (query heads of a key head times
 * nodes) a probability is multiplied with the scale of a block of values before it is rounded to bf16: blocks whose largest magnitude is
 * below 2^-80 may lose bits, and below 2^-110 may count as zero; above 2^97 that product may be infinite, which makes the block's zeros
 * NaN too.
 */
size_t i_attend_quantised_workspace(const i_attend_tree_problem* problem, int64_t bits);
int i_attend_quantised(const i_attend_tree_problem* problem, const i_attend_tensor* q, const i_quantised_cache* cache, const i_attend_tensor* o,
                       float* lse, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
