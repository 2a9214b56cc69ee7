// A cache whose rows are kept in 8 or 4 bits: what a row becomes, writing tokens and reading them back.
//
// A row of d columns, padded with zeros to a multiple of 32, is kept as blocks of 32 columns with a scale 2^(byte - 127) each.  4 bits:
// the numbers 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives; 8 bits: sign, 4 bits of exponent, 3 of fraction, 448 at most.
// The scale is the smallest power of two s with max |x| <= 7 s (4 bits) or 464 s (8 bits): then no element lies further
// above the largest number than half of the step below it.  x / s is exact, so a code is the number nearest to x / s, of two equally
// near ones the even code, with no rounding before it: the conversion instructions of the chip, which divide by the scale
// themselves.  Read back, a code times its scale is exact in bf16 (at most 4 significant bits), down to the least scale that is given,
// whose smallest number is 2^-126.  A block that holds a NaN, an infinity or a magnitude above 1.75 2^127 (whose nearest number may not
// be finite) gets scale 255 and reads as NaN.
//
// Bound by memory.  A lane has 8 columns, 4 lanes a block: 16-byte reads of bf16, and 4 or 8 bytes of codes.  (Two rows a thread with their
// loads ahead: 8 x 8 heads of 8192 x 128 read back 64 -> 74 us.)
#pragma once
#include "attend_tree.h"
#include "quantised_params.h"

namespace attend {

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;

constexpr uint32_t kNoNumber = 255;  // scale byte of a block that is NaN

template <int BITS>
struct Format {
  static_assert(BITS == 4 || BITS == 8, "bits");
  static constexpr int BYTES = 32 * BITS / 8;              // of a block's codes
  static constexpr int TOP = BITS == 4 ? 2 : 8;            // exponent of the largest number
  static constexpr uint32_t BEYOND = BITS == 4 ? 0x600000u : 0x680000u;  // fraction bits of 1.75 and 1.8125: 7 / 4, 464 / 256
  static constexpr int LEAST = BITS == 4 ? 2 : 10;         // least byte of a scale
};

// a block's scale from the bits of its largest magnitude
template <int BITS>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top > 0x7f600000u) return kNoNumber;
  const int byte = (int)(top >> 23) - Format<BITS>::TOP + ((top & 0x7fffffu) > Format<BITS>::BEYOND ? 1 : 0);
  return (uint32_t)max(byte, Format<BITS>::LEAST);
}
// ... as a number that conversions take
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte == kNoNumber ? 0x7fc00000u : byte << 23); }

// 8 columns, as 4 or 8 bytes of codes
__device__ __forceinline__ uint32_t encode4(const float (&x)[8], float scale) {
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
}
__device__ __forceinline__ uint32_t encode8(float a, float b, float c, float d, float scale) {
  s16x2 codes = {0, 0};
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(codes, a, b, scale, false);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(codes, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, codes);
}

// Codes back: 8 columns as bf16 (exact) or f32.
template <int BITS>
__device__ __forceinline__ bf16x8 decode(const uint32_t* codes, float scale, bf16_t) {
  bf16x2 p[4];
  if constexpr (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[0], scale, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[0], scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[0], scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[1], scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[1], scale, true);
  }
  return bf16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}
template <int BITS>
__device__ __forceinline__ f32x8 decode(const uint32_t* codes, float scale, float) {
  f32x2 p[4];
  if constexpr (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], scale, true);
  }
  return f32x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

__device__ __forceinline__ uint32_t divided(uint32_t x, uint32_t magic, uint32_t shift) { return (uint32_t)(((uint64_t)x * magic) >> shift); }

// A row of the tokens' operands (LPR lanes each, heads of a token beside each other) and its place in the cache.
struct MovedRow {
  uint32_t batch, head, token;
  bool there;        // a row of the operands
  bool live;         // a token that counts, with a slot in the sequence's pages
  int64_t page;      // -1: a page that the cache does not have
  uint32_t slot;
  __device__ __forceinline__ MovedRow(const QuantisedMoveParams& p, uint32_t lanes) {
    const uint32_t row = (blockIdx.y << kMoveAcross | blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
    there = row < p.rows;
    const uint32_t inside = there ? row : 0, of_batch = divided(inside, p.head_magic, p.head_shift);
    head = inside - of_batch * p.hkv;
    batch = divided(of_batch, p.token_magic, p.token_shift);
    token = of_batch - batch * p.n;
    const int64_t at = (int64_t)(p.first ? p.first[batch] : 0) + token;
    live = there && at >= 0 && at < p.slots && (!p.counts || (int)token < p.counts[batch]);
    const uint32_t inside_at = live ? (uint32_t)at : 0, index = divided(inside_at, p.page_magic, p.page_shift);
    slot = inside_at - index * p.page;
    const uint32_t listed = !live ? 0 : p.table ? (uint32_t)p.table[(int64_t)batch * p.table_stride + index] : batch;
    page = listed < p.pages ? (int64_t)listed : -1;
  }
  __device__ __forceinline__ uint8_t* codes(const QuantisedSide& s, int64_t page) const { return s.codes + page * s.page + head * s.head + slot * s.slot; }
  __device__ __forceinline__ uint8_t* scales(const QuantisedSide& s, int64_t page) const {
    return s.scales + page * s.scale_page + head * s.scale_head + slot * s.scale_slot;
  }
  template <typename T>
  __device__ __forceinline__ T* operand(const AttendOperand& x) const {
    return (T*)x.data + (int64_t)batch * x.sb + (int64_t)head * x.sh + (int64_t)token * x.sn;
  }
};

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));
}

template <typename T, int BITS, int LPR>
__device__ __forceinline__ void store_body(const QuantisedMoveParams& p) {
  const uint32_t lane = threadIdx.x % LPR, column = 8 * lane;
  const MovedRow row(p, LPR);
  const bool writes = row.live && row.page >= 0 && column < (p.d + 31) / 32 * 32;
  Frag<T> x[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    x[s] = zero_frag<T>();
    if (writes && column < p.d) x[s] = load_frag<T>(row.operand<const T>(s ? p.v : p.k) + column);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const QuantisedSide& side = s ? p.v_cache : p.k_cache;
    float y[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = (float)x[s][e];
      top = max(top, __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu);
    }
    // (the block's four lanes are four of a row's, none of them without the others; magnitudes order as their bits do, NaN above all)
    const uint32_t byte = scale_byte<BITS>(quad_max(top));
    if (!writes) continue;
    const float scale = byte == kNoNumber ? 1.0f : scale_of(byte);
    if (byte == kNoNumber) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = 0.0f;
    }
    uint8_t* codes = row.codes(side, row.page);
    if constexpr (BITS == 4) {
      *reinterpret_cast<uint32_t*>(codes + 4 * lane) = encode4(y, scale);
    } else {
      *reinterpret_cast<u32x2*>(codes + 8 * lane) = u32x2{encode8(y[0], y[1], y[2], y[3], scale), encode8(y[4], y[5], y[6], y[7], scale)};
    }
    if (lane % 4 == 0) row.scales(side, row.page)[lane / 4] = (uint8_t)byte;
  }
}

template <typename T, int BITS, int LPR>
__device__ __forceinline__ void load_body(const QuantisedMoveParams& p) {
  const uint32_t lane = threadIdx.x % LPR, column = 8 * lane;
  const MovedRow row(p, LPR);
  if (!row.there || column >= p.d) return;
  uint32_t codes[2][BITS / 4], byte[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const QuantisedSide& side = s ? p.v_cache : p.k_cache;
#pragma unroll
    for (int w = 0; w < BITS / 4; ++w) codes[s][w] = 0;
    byte[s] = 0;
    if (!row.live) continue;
    const int64_t page = max(row.page, (int64_t)0);
    const uint8_t* from = row.codes(side, page) + BITS * lane;
    if constexpr (BITS == 4) {
      codes[s][0] = *reinterpret_cast<const uint32_t*>(from);
    } else {
      const u32x2 both = *reinterpret_cast<const u32x2*>(from);
      codes[s][0] = both[0];
      codes[s][1] = both[1];
    }
    byte[s] = row.scales(side, page)[lane / 4];
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    Frag<T> x = decode<BITS>(codes[s], scale_of(byte[s] == kNoNumber ? 127 : byte[s]), T());
    if (byte[s] == kNoNumber) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (T)__builtin_nanf("");
    }
    T* to = row.operand<T>(s ? p.v : p.k) + column;
    if constexpr (sizeof(T) == 4) {
      store4(to, f32x4{x[0], x[1], x[2], x[3]});
      store4(to + 4, f32x4{x[4], x[5], x[6], x[7]});
    } else {
      *reinterpret_cast<Frag<T>*>(to) = x;
    }
  }
}

}  // namespace attend
