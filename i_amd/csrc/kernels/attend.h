// What the attention kernels with masks share: operand fragments, tiles in LDS, scores, running softmax.
//
// All products run on 16 x 16 matrix instructions.  Lane (r = lane & 15, g = lane >> 4) of a fragment holds the 8 elements
// 8 g .. 8 g + 7 of a 32-wide slab of row r (A operand) or column r (B operand); an accumulator holds rows 4 g .. 4 g + 3 of
// column r.  bf16: one v_mfma_f32_16x16x32 takes a fragment pair.  f32: eight v_mfma_f32_16x16x4 take its elements one by one
// (which four k a step adds up does not matter as long as both operands agree), so the kernels are the same text for both.
//
// A product whose left operand is a product's result needs no exchange between lanes: the two accumulators of 32 rows, rounded
// in order, are a B fragment whose k index runs 16 t + 4 g + i (t, i: element 4 t + i); the A operand of that second product is
// read from LDS transposed with the same order of k.
//
// Tiles reach LDS by 16-byte transfers that bypass the registers (dma16).  Rows are 128, 256, 512 or 1024 bytes; the 16-byte
// chunk c of row w lies at chunk c ^ swizzle(w), so that 16 rows read at one chunk, and 16 rows read at a pair of chunks
// (transposed reads), spread over the 256-byte window of the banks.
#pragma once
#include <type_traits>

#include "attend_params.h"
#include "common.h"

namespace attend {

typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

template <typename T>
using Frag = std::conditional_t<std::is_same_v<T, float>, f32x8, bf16x8>;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// Results of matrix instructions on their way to vector instructions beyond a branch.  A vector instruction may read such a result
// no sooner than 8 (bf16) or 10 (f32) wait states after it was issued.  The compiler fills them in, but not all of them where a branch
// lies between (one kernel gave wrong sums; the build reads the assembly for such pairs).  Here they are spelled out: every
// result passes the first row of statements, all matrix instructions lie before its end, and every result passes the second.
template <typename T, int N>
__device__ __forceinline__ void settle(f32x4 (&s)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(s[n]));
  if constexpr (std::is_same_v<T, float>) asm volatile("s_nop 9" : "+v"(s[0]));
  else asm volatile("s_nop 7" : "+v"(s[0]));
#pragma unroll
  for (int n = 1; n < N; ++n) asm volatile("" : "+v"(s[n]));
}

// Addition to an accumulator that lives in the accumulation registers for a whole kernel.  bf16: spelled out, since the compiler moves
// accumulators between the two register files when a wavefront has more than 256 registers' worth (grad_keys at d = 128: a quarter of
// its instructions).  The right operands are ready()'d first (two wait states between a vector instruction that writes an operand
// and the matrix instruction that reads it), the left ones come from LDS; sums are read after settled().
__device__ __forceinline__ void add_mma(f32x4& c, bf16x8 a, bf16x8 b) {
  asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void add_mma(f32x4& c, f32x8 a, f32x8 b) { c = mma(a, b, c); }
// Product with a right operand that lives in the accumulation registers for a whole kernel, sum in vector registers: the compiler
// copies such an operand before every use.  first: no addend.  The sum is read after settle().
__device__ __forceinline__ void mma_kept(f32x4& c, bf16x8 a, const bf16x8& b, bool first) {
  if (first) asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=v"(c) : "v"(a), "a"(b));
  else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
}
__device__ __forceinline__ void mma_kept(f32x4& c, f32x8 a, const f32x8& b, bool first) { c = mma(a, b, first ? f32x4{0, 0, 0, 0} : c); }
template <int N>
__device__ __forceinline__ void keep(bf16x8 (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+a"(x[n]));
}
template <int N>
__device__ __forceinline__ void keep(f32x8 (&)[N]) {}
template <typename F, int N>
__device__ __forceinline__ void ready(F (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("s_nop 1" : "+v"(x[n]));
}
// sums for add_mma, zero.  (Through the asm, since the compiler takes apart a vector that enters a loop as a constant, and then keeps
// its elements in vector registers between two trips.)
template <typename T, int N, int M>
__device__ __forceinline__ void clear_sums(f32x4 (&c)[N][M]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      c[n][m] = f32x4{0, 0, 0, 0};
      if constexpr (!std::is_same_v<T, float>) asm volatile("" : "+a"(c[n][m]));
    }
}
// the wait between the last add_mma and the first instruction that reads a sum
template <typename T, int N, int M>
__device__ __forceinline__ void settled(f32x4 (&c)[N][M]) {
  if constexpr (std::is_same_v<T, float>) return;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int m = 0; m < M; ++m) asm volatile("s_nop 7" : "+a"(c[n][m]));
}

// Operands loaded before a loop and used in it are waited for here.  Left to the loop, the compiler's wait for them stands inside it
// and takes the requested tiles with it on every trip: it does not know of those (a quarter of the forward kernel's time at 4096 keys).
template <typename F, int N>
__device__ __forceinline__ void arrive(F (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[n]));
}

// the four 16-lane groups' copies of a value put together, result in all of them
__device__ __forceinline__ void both_rows(float x, float& lo, float& hi) {
  float a = x, b = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  lo = a;
  hi = b;
}
__device__ __forceinline__ float groups_max(float x) {
  float lo, hi;
  both_rows(x, lo, hi);
  return half_max(fmaxf(lo, hi));
}
__device__ __forceinline__ float groups_sum(float x) {
  float lo, hi;
  both_rows(x, lo, hi);
  return half_sum(lo + hi);
}

// the sum over 16 consecutive lanes, in all of them
__device__ __forceinline__ float row_sum(float x) {
  auto turned = [](float y, auto control) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), decltype(control)::value, 0xf, 0xf, false)); };
  x += turned(x, std::integral_constant<int, 0x121>{});
  x += turned(x, std::integral_constant<int, 0x122>{});
  x += turned(x, std::integral_constant<int, 0x124>{});
  return x + turned(x, std::integral_constant<int, 0x128>{});
}

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
  Frag<T> z;
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = (T)0.0f;
  return z;
}

// 8 consecutive elements, 16-byte aligned
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* at) {
  if constexpr (std::is_same_v<T, float>) {
    const u32x4 lo = ldg128(at), hi = ldg128(at + 4);
    return __builtin_bit_cast(f32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    return __builtin_bit_cast(bf16x8, ldg128(at));
  }
}

__device__ __forceinline__ void store4(float* at, f32x4 x) { *reinterpret_cast<f32x4*>(at) = x; }
__device__ __forceinline__ void store4(bf16_t* at, f32x4 x) {
  bf16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (bf16_t)x[e];
  *reinterpret_cast<bf16x4*>(at) = y;
}

// DPAD: columns of a row in LDS (a power of two); ROWS rows.
template <typename T, int DPAD, int ROWS>
struct Tile {
  static constexpr int RB = DPAD * (int)sizeof(T);        // bytes per row
  static constexpr int CH = RB / 16;                      // chunks per row
  static constexpr int RPB = RB >= 256 ? 1 : 256 / RB;    // rows per bank window
  static constexpr int SW = 16 / RPB;                     // values of the swizzle
  static constexpr int RPW = 1024 / RB;                   // rows per wave-load
  static constexpr int BYTES = ROWS * RB;
  static constexpr int WL = BYTES / 1024;                 // wave-loads
  static_assert(RB >= 128 && RB <= 1024 && BYTES % 1024 == 0, "row size");
  // What the 16-byte chunks of a row are XOR-ed with: a linear map of the row's bits, so that 16 lanes that LDS serves together (64
  // banks, 256 bytes) meet no bank twice.  A read of 16 bytes a lane is served in groups of 16 lanes: rows 0-3 and 12-15 of one
  // chunk with rows 4-11 of its neighbour; so the row difference that maps to 1 may not tell these two apart.
  //   f32, transposed: rows g, 4 + g, 8 + g, 12 + g of a 64-byte group together: the row's bits as they are.
  //   bf16, transposed: rows 0-7 (8-15) of a 32-byte group together: the difference that maps to 1 lies in the top bit too.
  // (Counted: no conflicts, where the row's bits as they are cost bf16 two turns a transposed read, and one place up four a row read.)
  static constexpr __device__ __forceinline__ uint32_t swizzle(uint32_t row) {
    const uint32_t x = (row / RPB) % SW, top = x / (SW / 2), next = x / (SW / 4) % 2;
    return std::is_same_v<T, float> ? x : 2 * (x % (SW / 4)) | (top ^ next) * (SW / 2) | top;
  }

  // Requests of tiles of a matrix whose rows lie `stride` bytes apart, by NW wavefronts.  `chunks` of a row exist in memory;
  // the others are left as they are (zeros).
  template <int NW>
  struct Requests {
    static constexpr int EACH = (WL + NW - 1) / NW;  // wave-loads of a wavefront
    static constexpr int STEP = NW * RPW;            // rows between two of them
    uint32_t stride, chunks, row, chunk;             // of this lane in its wavefront's first one
    int wave;
    __device__ __forceinline__ Requests(uint32_t stride, uint32_t d, int wave, int lane) : stride(stride), chunks(d * (uint32_t)sizeof(T) / 16), wave(wave) {
      row = wave * RPW + lane / CH;
      chunk = (lane % CH) ^ swizzle(row);
    }
    // Rows row0 .. row0 + ROWS; a row outside lo .. hi - 1 is read as the nearest one inside.
    __device__ __forceinline__ void operator()(const char* base, int row0, int lo, int hi, uint32_t lds) const {
      if (WL < NW && wave >= WL) return;
      const char* at = base + (int64_t)row0 * stride;
      const uint32_t to = lds + wave * 1024;
      if (row0 >= lo && row0 + ROWS <= hi) {
        // all in place: what changes between wave-loads is scalar, but for a constant XOR where the swizzle's period is longer
        if (chunks == CH) {
#pragma unroll
          for (int it = 0; it < EACH; ++it)
            dma16(at + (int64_t)(it * STEP) * stride, row * stride + 16 * (chunk ^ swizzle(it * STEP)), to + it * NW * 1024);
        } else {
#pragma unroll
          for (int it = 0; it < EACH; ++it)
            if ((chunk ^ swizzle(it * STEP)) < chunks)
              dma16(at + (int64_t)(it * STEP) * stride, row * stride + 16 * (chunk ^ swizzle(it * STEP)), to + it * NW * 1024);
        }
      } else {
#pragma unroll
        for (int it = 0; it < EACH; ++it) {
          const uint32_t c = chunk ^ swizzle(it * STEP);
          const int key = min(max(row0 + (int)row + it * STEP, lo), hi - 1);
          if (c < chunks) dma16(at, (uint32_t)(key - row0) * stride + 16 * c, to + it * NW * 1024);
        }
      }
    }
  };
};

// Reads of operands from a tile: rows (A operand, 8 consecutive columns a lane) and transposed.
template <typename T, int DPAD>
struct Reader {
  using L = Tile<T, DPAD, 32>;
  uint32_t row_at;    // this lane's place in a 16-row block, slab 0
  uint32_t across_at[std::is_same_v<T, float> ? 4 : 1];

  __device__ __forceinline__ explicit Reader(int lane) {
    const uint32_t r = lane & 15, g = lane >> 4;
    if constexpr (std::is_same_v<T, float>) {
      row_at = r * L::RB + 16 * ((2 * g) ^ L::swizzle(r));
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) across_at[i] = (4 * g + i) * L::RB + 16 * ((r >> 2) ^ L::swizzle(4 * g + i)) + 4 * (r & 3);
    } else {
      row_at = r * L::RB + 16 * (g ^ L::swizzle(r));
      // lane 4 j + q of a 16-lane block points at row 4 g + j, columns 4 q .. 4 q + 3
      const uint32_t row = 4 * g + (r >> 2), q = r & 3;
      across_at[0] = row * L::RB + 16 * ((q >> 1) ^ L::swizzle(row)) + 8 * (q & 1);
    }
  }
  // rows 16 block .. + 16, columns 32 slab .. + 32
  __device__ __forceinline__ Frag<T> rows(const char* tile, int block, int slab) const {
    const char* at = tile + 16 * block * L::RB;
    if constexpr (std::is_same_v<T, float>) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(at + (row_at ^ (128 * slab)));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(at + (row_at ^ (128 * slab + 16)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const bf16x8*>(at + (row_at ^ (64 * slab)));
    }
  }
  // columns 16 block .. + 16 as rows, rows 32 group .. + 32 as k in the order of an accumulator pair
  __device__ __forceinline__ Frag<T> across(const char* tile, int block, int group) const {
    const char* at = tile + 32 * group * L::RB;
    if constexpr (std::is_same_v<T, float>) {
      f32x8 x;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * t + i] = *reinterpret_cast<const float*>(at + 16 * t * L::RB + (across_at[i] ^ (64 * block)));
      return x;
    } else {
      const char* here = at + (across_at[0] ^ (32 * block));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(here));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(here + 16 * L::RB));
      return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Scores from products, in the base-2 domain of the exponentials (1 / ln 2 times the score).  Where there is neither cap nor bias
// that factor is left to the exponential's own multiply-add (mult), else `all` applies it.
//
// A cap is x = cap tanh(y), y = scale s / cap.  For |y| <= 3/8 tanh(y) is y times a polynomial of degree 3 in y^2, by
// interpolation at the Chebyshev points of [0, 9/64]: off by at most 1.2e-7 of its value, five instructions a score and one more to see
// that it will do.  Beyond it is 1 - 2 / (e^{2y} + 1), right at both ends (e^{2y} = 0 or infinite), whose cancellation costs two bits at
// 3/8 and whose two transcendental instructions take four turns each.  Scores are mostly far below their cap, so a wavefront
// looks at the largest of its tile first and takes the polynomial alone where it can.
struct Bend {
  float mult;      // what the exponential multiplies by: 1 when bent
  float into;      // capped: product -> y; else product -> score
  float small2;    // capped: squared product of y = 3/8
  float cap2;      // cap / ln 2
  float back;      // capped: 1 / cap2 (score -> tanh, for the gradient)
  float c[4];      // capped: the polynomial, in squares of the product, times the score's factor
  bool capped, bent;
  static constexpr float I_LOG2_E = 1.44269504089f;
  __device__ __forceinline__ Bend(float scale, float cap, bool biased) {
    capped = cap > 0.0f;
    // (a zero scale is applied on its own: 0 times the -inf of a masked score would be no number)
    bent = capped || biased || !(scale > 0.0f);
    mult = bent ? 1.0f : scale * I_LOG2_E;
    into = capped ? scale / cap : scale * I_LOG2_E;
    small2 = 0.140625f / (into * into);
    cap2 = cap * I_LOG2_E;
    back = capped ? 1.0f / cap2 : 0.0f;
    const float y2 = into * into, factor = scale * I_LOG2_E;
    constexpr float tanh_over_y[4] = {0.99999994f, -0.333319711f, 0.132844312f, -0.0482689079f};
    float power = factor;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      c[n] = tanh_over_y[n] * power;
      power *= y2;
    }
    // a cap so far below the scores that a coefficient overflows (a product of 0 would give 0 times infinity): never the polynomial
    if (!__builtin_isfinite(c[3])) small2 = -1.0f;
  }
  // |y| <= 3/8: score over product, from the product's square
  __device__ __forceinline__ float small(float u) const {
    return __builtin_fmaf(u, __builtin_fmaf(u, __builtin_fmaf(u, c[3], c[2]), c[1]), c[0]);
  }
  __device__ __forceinline__ float large(float s) const {
    return cap2 - 2.0f * cap2 * __builtin_amdgcn_rcpf(fast_exp2(s * into * (2.0f * I_LOG2_E)) + 1.0f);
  }
  // whether the polynomial will do for all of a wavefront's products (N x M vectors)
  template <int N, int M>
  __device__ __forceinline__ bool all_small(const f32x4 (&s)[N][M]) const {
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const f32x4 u = s[n][m] * s[n][m];
        most = fmaxf(fmaxf(most, fmaxf(u[0], u[1])), fmaxf(u[2], u[3]));
      }
    return __builtin_amdgcn_ballot_w64(!(most <= small2)) == 0;
  }
  // products into scores
  template <int N, int M>
  __device__ __forceinline__ void all(f32x4 (&s)[N][M]) const {
    if (!capped) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int m = 0; m < M; ++m) s[n][m] *= into;
    } else if (all_small(s)) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][m][i] *= small(s[n][m][i] * s[n][m][i]);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float u = s[n][m][i] * s[n][m][i], wide = large(s[n][m][i]);
            s[n][m][i] = u <= small2 ? s[n][m][i] * small(u) : wide;
          }
    }
  }
  template <int N>
  __device__ __forceinline__ void all(f32x4 (&s)[N]) const {
    all(reinterpret_cast<f32x4(&)[1][N]>(s));
  }
  // one product into the exponential's argument before bias and lse
  __device__ __forceinline__ float one(float s) const {
    if (!bent) return s * mult;
    if (!capped) return s * into;
    const float u = s * s;
    return u <= small2 ? s * small(u) : large(s);
  }
  // d score / d product over the scale, from the unbiased score
  __device__ __forceinline__ float slope(float x) const {
    const float t = x * back;
    return __builtin_fmaf(-t, t, 1.0f);
  }
};

// Keys that a query sees: first <= j < last.  Neither is negative, so that their difference is right whatever the bounds given are.
struct Span {
  int first, last;
};
__device__ __forceinline__ Span span_of(const AttendParams& p, uint32_t batch, uint32_t row) {
  Span s{0, (int)p.nk};
  if (p.first) s.first = max(p.first[(size_t)batch * p.nq + row], 0);
  if (p.last) s.last = min(p.last[(size_t)batch * p.nq + row], (int)p.nk);
  if (p.causal) s.last = min(s.last, (int)row + p.shift + 1);
  s.last = max(s.last, 0);
  return s;
}
// Of several queries: least and largest first, least and largest last.  A query that sees nothing widens neither first_least nor
// last_most, and makes every key tile one that has to be masked.
struct Spans {
  int first_least, first_most, last_least, last_most;
  __device__ __forceinline__ void none() {
    first_least = 0x7fffffff;
    first_most = 0;
    last_least = 0x7fffffff;
    last_most = 0;
  }
  __device__ __forceinline__ void add(Span s) {
    const bool sees = s.first < s.last;
    first_least = min(first_least, sees ? s.first : 0x7fffffff);
    last_most = max(last_most, sees ? s.last : 0);
    first_most = max(first_most, sees ? s.first : 0x7fffffff);
    last_least = min(last_least, sees ? s.last : 0);
  }
  __device__ __forceinline__ void add(const Spans& s) {
    first_least = min(first_least, s.first_least);
    first_most = max(first_most, s.first_most);
    last_least = min(last_least, s.last_least);
    last_most = max(last_most, s.last_most);
  }
  // over 16 consecutive lanes (rotations inside a row of lanes, which cost no LDS access), or all 64
  template <int CONTROL>
  __device__ __forceinline__ Spans moved() const {
    return Spans{__builtin_amdgcn_update_dpp(first_least, first_least, CONTROL, 0xf, 0xf, false), __builtin_amdgcn_update_dpp(first_most, first_most, CONTROL, 0xf, 0xf, false),
                 __builtin_amdgcn_update_dpp(last_least, last_least, CONTROL, 0xf, 0xf, false), __builtin_amdgcn_update_dpp(last_most, last_most, CONTROL, 0xf, 0xf, false)};
  }
  template <int LANES>
  __device__ __forceinline__ void over_lanes() {
    static_assert(LANES == 16 || LANES == 64, "lanes");
    add(moved<0x121>());
    add(moved<0x122>());
    add(moved<0x124>());
    add(moved<0x128>());
    if constexpr (LANES == 64) {
#pragma unroll
      for (int bit = 16; bit < 64; bit <<= 1) add(Spans{__shfl_xor(first_least, bit), __shfl_xor(first_most, bit), __shfl_xor(last_least, bit), __shfl_xor(last_most, bit)});
    }
  }
  __device__ __forceinline__ void uniform() {
    first_least = __builtin_amdgcn_readfirstlane(first_least);
    first_most = __builtin_amdgcn_readfirstlane(first_most);
    last_least = __builtin_amdgcn_readfirstlane(last_least);
    last_most = __builtin_amdgcn_readfirstlane(last_most);
  }
  __device__ __forceinline__ bool touches(int k0, int k1) const { return k0 < last_most && k1 > first_least; }
  __device__ __forceinline__ bool whole(int k0, int k1) const { return k0 >= first_most && k1 <= last_least; }
};

// 16 QB query columns of a wavefront and their running softmax:  O^T = sum_j V_j^T p_j, kept relative to 2^m.
//
// Where every score of a tile counts as it is (no mask, no bias) no maximum is taken while things go well: the probabilities are
// computed against the reference m that a query already has, and only if some lane's sum over the tile is not below 2^30, or a query
// has no reference yet, the tile is computed again, from its products on, the other way: there a reference moves to the tile's
// maximum when that passes it by 8 (in the exponent), and sum and output are corrected.  Floating point is scale-free, so that any
// reference gives the same result while nothing overflows.  The sum is taken over the f32 probabilities, lane by lane, and put
// together once.  bf16: the probabilities are rounded to bf16 for the second product, whose other operand has no more bits than that.
template <typename T, int DPAD, int DUSE, int QB>
struct Rows {
  static constexpr int KS = DUSE / 32, DT = DUSE / 16;
  Frag<T> q[QB][KS];
  f32x4 o[QB][DT];
  float m[QB], l[QB];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int b = 0; b < QB; ++b) {
#pragma unroll
      for (int t = 0; t < DT; ++t) o[b][t] = f32x4{0, 0, 0, 0};
      m[b] = -INFINITY;
      l[b] = 0.0f;
    }
  }
  __device__ __forceinline__ void load_q(int b, const T* row, bool there, uint32_t d, int g) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t at = 32 * ks + 8 * g;
      q[b][ks] = there && at < d ? load_frag<T>(row + at) : zero_frag<T>();
    }
  }
  // S^T of a tile of 16 KT keys
  template <int KT>
  __device__ __forceinline__ void products(f32x4 (&s)[QB][KT], const Reader<T, DPAD>& reader, const char* tile) const {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int b = 0; b < QB; ++b) s[b][kt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const Frag<T> a = reader.rows(tile, kt, ks);
#pragma unroll
        for (int b = 0; b < QB; ++b) s[b][kt] = mma(a, q[b][ks], s[b][kt]);
      }
    }
    settle<T>(reinterpret_cast<f32x4(&)[QB * KT]>(s));
  }
  // Probabilities of a tile against the references that there are, exp2(exponent(score, reference)); false: they will not do.
  template <int KT, typename Exponent>
  __device__ __forceinline__ bool weigh(const f32x4 (&s)[QB][KT], Exponent exponent, Frag<T> (&pf)[QB][KT / 2], float (&sum)[QB]) const {
    bool good = true;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const float ref = m[b] == -INFINITY ? 0.0f : m[b];
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(exponent(s[b][kt][i], ref));
          part[i & 1] += e;
          pf[b][kt / 2][4 * (kt & 1) + i] = (T)e;
        }
      sum[b] = part[0] + part[1];
      good = good && sum[b] < 0x1p30f && m[b] > -INFINITY;
    }
    return __builtin_amdgcn_ballot_w64(!good) == 0;
  }
  // The largest of a tile's scores as reference where it passes the old one by 8.  (A query that has seen nothing keeps -inf: its
  // scores are -inf and weigh 0 on 0.)
  template <int KT>
  __device__ __forceinline__ void move(const f32x4 (&s)[QB][KT]) {
    bool far = false;
    float top[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      top[b] = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[b] = fmaxf(top[b], s[b][kt][i]);
      far = far || top[b] > m[b] + 8.0f;
    }
    if (__builtin_amdgcn_ballot_w64(far) == 0) return;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const float now = fmaxf(m[b], groups_max(top[b]));
      const float keep = m[b] == -INFINITY ? 0.0f : fast_exp2(m[b] - now);
      m[b] = now;
      l[b] *= keep;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[b][t] *= keep;
    }
  }
  // One tile of 16 KT keys.  `plain`: every query of the wavefront sees every key and there is no bias; else finish(s) turns bent
  // products into scores.
  template <int KT, typename Finish>
  __device__ __forceinline__ void tile(const char* k, const char* v, const Bend& bend, bool plain, Finish finish, const Reader<T, DPAD>& reader) {
    f32x4 s[QB][KT];
    Frag<T> pf[QB][KT / 2];
    float sum[QB];
    products(s, reader, k);
    bool done = false;
    if (plain) {
      if (!bend.bent) done = weigh(s, [&](float x, float ref) { return __builtin_fmaf(x, bend.mult, -ref); }, pf, sum);
      else if (bend.capped && bend.all_small(s)) done = weigh(s, [&](float x, float ref) { return __builtin_fmaf(x, bend.small(x * x), -ref); }, pf, sum);
      if (!done) products(s, reader, k);
    }
    if (!done) {
      if (bend.bent) {
        bend.all(s);
      } else {
#pragma unroll
        for (int b = 0; b < QB; ++b)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) s[b][kt] *= bend.mult;
      }
      finish(s);
      move(s);
      weigh(s, [](float x, float ref) { return x - ref; }, pf, sum);
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) l[b] += sum[b];
#pragma unroll
    for (int u = 0; u < KT / 2; ++u)
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const Frag<T> a = reader.across(v, t, u);
#pragma unroll
        for (int b = 0; b < QB; ++b) o[b][t] = mma(a, pf[b][u], o[b][t]);
      }
  }
};

// The results of NW wavefronts that saw different keys of the same 16 QB rows, put together through their tile memory (`mine` of
// each, 16 QB x DPAD f32, 16-byte chunk c of row w at chunk c ^ (w & 15)).  give(row, column, four outputs, lse base 2) for every four
// columns.
template <int NW, int QB>
struct Merge {
  float m[NW][16 * QB], l[NW][16 * QB];
};
template <typename T, int DPAD, int DUSE, int NW, int QB, typename Give>
__device__ __forceinline__ void merge_rows(const Rows<T, DPAD, DUSE, QB>& rows, Merge<NW, QB>& shared, char* tiles, int tile_bytes, uint32_t d, uint32_t count, Give give) {
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4, wave = tid >> 6;
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(tiles + wave * tile_bytes);
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const float sum = groups_sum(rows.l[b]);
    if (g == 0) {
      shared.m[wave][16 * b + r] = rows.m[b];
      shared.l[wave][16 * b + r] = sum;
    }
#pragma unroll
    for (int t = 0; t < DUSE / 16; ++t) store4(mine + (16 * b + r) * DPAD + 4 * ((4 * t + g) ^ r), rows.o[b][t]);
  }
  __syncthreads();
  const uint32_t fours = d / 4;
  for (uint32_t i = tid; i < count * fours; i += 64 * NW) {
    const uint32_t row = i / fours, c = i - row * fours;
    float top = shared.m[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, shared.m[w][row]);
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = shared.m[w][row], weigh = m == -INFINITY ? 0.0f : fast_exp2(m - top);
      sum += weigh * shared.l[w][row];
      // (a wavefront that had no tile leaves zeros)
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tiles + w * tile_bytes) + row * DPAD + 4 * (c ^ (row & 15))) * weigh;
    }
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    give(row, 4 * c, o, top == -INFINITY ? -INFINITY : top + __builtin_amdgcn_logf(sum));
  }
}

// `total` pieces of work dealt out in equal runs, of which the first ones have one more where they do not divide evenly.
struct Deal {
  uint32_t shares, each, more;
  __device__ __forceinline__ Deal(uint32_t total, uint32_t most) : shares(min(most, max(total, 1u))), each(total / shares), more(total - each * shares) {}
  __device__ __forceinline__ uint32_t begin(uint32_t share) const { return share * each + min(share, more); }
  // the share that has a piece
  __device__ __forceinline__ uint32_t of(uint32_t piece) const {
    const uint32_t longer = more * (each + 1);
    return piece < longer ? piece / (each + 1) : more + (piece - longer) / max(each, 1u);
  }
};

// Keys of a tile that nobody sees, between keys that are seen, may hold anything: their probability of zero must not meet what is
// no number.  Where a tile may have such keys their rows are set to zero in LDS before the product that takes them as addends: found
// from the queries' intervals (a tree: from the nodes' words), as a bit for each of 64 keys.  What a wavefront does about its own tiles needs
// no barrier; a shared tile is left to all threads between two barriers, only where it has such a key.  Where they may lie is found
// out once (Gap), and only tiles there are looked at: documents, windows and prefixes cost nothing (looked at in every partly seen
// tile: 68 -> 77 us for documents of 6001 tokens), documents of 300 with 20 of padding between them 32.0 -> 33.8 us.
__device__ __forceinline__ uint64_t seen_keys(Span s, int k0) {
  const int lo = min(max(s.first - k0, 0), 64), hi = min(max(s.last - k0, 0), 64);
  return (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 64 ? ~0ull : (1ull << lo) - 1);
}
__device__ __forceinline__ uint32_t row_or(uint32_t bits) {
  int x = (int)bits;
  x |= __builtin_amdgcn_update_dpp(x, x, 0x121, 0xf, 0xf, false);
  x |= __builtin_amdgcn_update_dpp(x, x, 0x122, 0xf, 0xf, false);
  x |= __builtin_amdgcn_update_dpp(x, x, 0x124, 0xf, 0xf, false);
  x |= __builtin_amdgcn_update_dpp(x, x, 0x128, 0xf, 0xf, false);
  return (uint32_t)x;
}
__device__ __forceinline__ uint64_t wave_or(uint64_t bits) {
  const int lo = (int)row_or((uint32_t)bits), hi = (int)row_or((uint32_t)(bits >> 32));
  uint64_t all = 0;
#pragma unroll
  for (int at = 0; at < 64; at += 16) all |= (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, at) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, at);
  return all;
}
// (Nothing of this rare path is computed ahead of a loop: it would cost the loop's registers, up to 12.  So the lane is asked for anew.)
__device__ __forceinline__ int lane_now() {
  int lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}
// Where keys lie that nobody sees, between seen ones: a query's interval on either side of such a key, some two that follow one another (but
// for queries that see nothing) have it between them.  None: lo > hi.
struct Gap {
  int lo, hi;
  __device__ __forceinline__ bool touches(int k0, int k1) const { return k0 < hi && k1 > lo; }
};
__device__ __forceinline__ void widen(Spans& gap, Span a, Span b) {
  const int lo = min(a.last, b.last), hi = max(a.first, b.first);
  gap.first_least = min(gap.first_least, lo < hi ? lo : 0x7fffffff);
  gap.last_most = max(gap.last_most, lo < hi ? hi : 0);
}
// between the intervals of `count` queries
__device__ __forceinline__ Gap gap_between(const Span* of, int count) {
  Spans gap;
  gap.none();
  Span before{0, 0};
  const int lane = lane_now();
  for (int n0 = 0; n0 < count; n0 += 64) {
    const Span mine = of[min(n0 + lane, count - 1)];
    const bool sees = n0 + lane < count && mine.first < mine.last;
    const uint64_t seeing = __builtin_amdgcn_ballot_w64(sees), after = seeing >> lane >> 1;
    if (sees && after) widen(gap, mine, of[n0 + lane + 1 + __builtin_ctzll(after)]);
    if (seeing == 0) continue;
    const int least = __builtin_ctzll(seeing), most = 63 - __builtin_clzll(seeing);
    const Span begin{__builtin_amdgcn_readlane(mine.first, least), __builtin_amdgcn_readlane(mine.last, least)};
    if (before.first < before.last) widen(gap, before, begin);
    before = Span{__builtin_amdgcn_readlane(mine.first, most), __builtin_amdgcn_readlane(mine.last, most)};
  }
  if (__builtin_amdgcn_ballot_w64(gap.last_most > 0) == 0) return Gap{0x7fffffff, 0};
  gap.over_lanes<64>();
  gap.uniform();
  return Gap{gap.first_least, gap.last_most};
}
// ... of 16, one in each of the first 16 lanes (and again in the others)
__device__ __forceinline__ Gap gap_between(Span mine) {
  Spans gap;
  gap.none();
  const int lane = lane_now() & 15;
  const uint32_t seeing = (uint32_t)__builtin_amdgcn_ballot_w64(mine.first < mine.last) & 0xffffu, after = seeing >> lane >> 1;
  const int next = after ? lane + 1 + __builtin_ctz(after) : lane;
  const Span other{__shfl(mine.first, next), __shfl(mine.last, next)};
  if (after && mine.first < mine.last) widen(gap, mine, other);
  if (__builtin_amdgcn_ballot_w64(gap.last_most > 0) == 0) return Gap{0x7fffffff, 0};
  gap.over_lanes<16>();
  gap.uniform();
  return Gap{gap.first_least, gap.last_most};
}
// of keys k0 .. k0 + KEYS - 1 those that `count` queries leave out between lo and hi
template <int KEYS>
__device__ __forceinline__ uint64_t unseen_keys(const Span* of, int count, int k0, int lo, int hi) {
  static_assert(KEYS <= 64, "a bit each");
  uint64_t seen = 0;
  for (int n = lane_now(); n < count; n += 64) seen |= seen_keys(of[n], k0);
  return seen_keys(Span{lo, min(hi, k0 + KEYS)}, k0) & ~wave_or(seen);
}
// rows of a tile whose bit is set: zeros, by NW wavefronts
template <typename L, int NW>
__device__ __forceinline__ void clear_rows(char* tile, uint64_t rows, int wave) {
  uint32_t zero = 0;
  asm volatile("" : "+v"(zero));
#pragma unroll 1
  for (int at = 64 * wave + lane_now(); at < L::BYTES / 16; at += 64 * NW)
    if (rows >> (at / L::CH) & 1) *reinterpret_cast<u32x4*>(tile + 16 * at) = u32x4{zero, zero, zero, zero};
}

// The workgroup's tile memory set to zero: what no transfer writes (the columns past d) then reads as zero.
template <int BYTES, int THREADS>
__device__ __forceinline__ void clear_tiles(char* lds, int tid) {
  for (int at = 16 * tid; at < BYTES; at += 16 * THREADS) *reinterpret_cast<u32x4*>(lds + at) = u32x4{0, 0, 0, 0};
}

}  // namespace attend
