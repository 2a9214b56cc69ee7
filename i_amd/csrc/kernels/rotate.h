// Norm and rotary position of every head of queries and keys in one pass, and its gradient.
//
//   n = x / sqrt(mean(x^2) + eps),   u = n w,   y = turn(u):  (u_a cos t - u_b sin t, u_b cos t + u_a sin t) for a pair of columns,
//   t = position(axis of the pair) * frequency of the pair
//   gradient:  g = turn back(dy),   dw = sum over rows of g n,   dx = (g w - n mean(g w n)) / sqrt(mean(x^2) + eps)
//
// Bound by memory: every row is read once and written once.  4, 8 or 16 lanes have a row, 16 columns each, so that a row's sum is two to
// four exchanges inside a row of lanes.  A workgroup has the tokens of one wavefront's rows (16, 8 or 4) and a run of heads, every
// wavefront each fourth head of it.  Cosines and sines of its tokens are computed once, two angles a thread, and handed over
// through LDS; lanes keep those of their columns for all heads of the run.  An angle costs a product and a remainder in 64 bits
// (positions reach millions, of which f32 would leave an angle no digit) and two polynomials.  Which 16 columns a lane has follows the pairs:
//   halves      (j, j + pairs), pairs a multiple of 8: two runs of 8 columns, `pairs` apart, so that a pair is in one lane
//   neighbours  (2 j, 2 j + 1): 16 columns in a row
//   apart       (j, j + pairs) with any other number of pairs: 16 columns in a row, partners through LDS
#pragma once
#include "common.h"
#include "rotate_params.h"

namespace rotate {

constexpr int kWaves = 4;
enum Kind { kHalves, kNeighbours, kApart };

template <int CONTROL>
__device__ __forceinline__ float moved(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CONTROL, 0xf, 0xf, false));
}
// the sum over LANES consecutive lanes (4, 8 or 16), the same bits in all of them
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
  x += moved<0xb1>(x);  // neighbour, and neighbour's pair
  x += moved<0x4e>(x);
  if constexpr (LANES >= 8) x += moved<0x141>(x);   // the other four of eight, mirrored
  if constexpr (LANES >= 16) x += moved<0x140>(x);  // the other eight
  return x;
}

// 8 elements as they lie in memory, and as f32
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  f32x4 lo, hi;
  __device__ __forceinline__ void load(const float* at) {
    lo = __builtin_bit_cast(f32x4, ldg128(at));
    hi = __builtin_bit_cast(f32x4, ldg128(at + 4));
  }
  __device__ __forceinline__ float operator[](int e) const { return e < 4 ? lo[e] : hi[e - 4]; }
};
template <>
struct Eight<bf16_t> {
  bf16x8 all;
  __device__ __forceinline__ void load(const bf16_t* at) { all = __builtin_bit_cast(bf16x8, ldg128(at)); }
  __device__ __forceinline__ float operator[](int e) const { return (float)all[e]; }
};

__device__ __forceinline__ void store8(float* at, const float (&x)[16], int from) {
  *reinterpret_cast<f32x4*>(at) = f32x4{x[from], x[from + 1], x[from + 2], x[from + 3]};
  *reinterpret_cast<f32x4*>(at + 4) = f32x4{x[from + 4], x[from + 5], x[from + 6], x[from + 7]};
}
__device__ __forceinline__ void store8(bf16_t* at, const float (&x)[16], int from) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (bf16_t)x[from + e];
  *reinterpret_cast<bf16x8*>(at) = v;
}

// The columns of a lane: `a` .. a + 7 and `b` .. b + 7, those that exist.
template <int KIND>
struct Columns {
  uint32_t a, b;
  bool has_a, has_b;
  __device__ __forceinline__ Columns(const RotateParams& p, uint32_t lane) {
    const uint32_t turning = KIND == kHalves ? p.pairs / 8 : 0;  // lanes whose two runs are a pair's halves
    const bool halves = lane < turning;
    const uint32_t rest = 8 * (2 * turning + 2 * (lane - turning));
    a = halves ? 8 * lane : rest;
    b = halves ? 8 * lane + p.pairs : rest + 8;
    has_a = a < p.d;
    has_b = b < p.d;
  }
  // a lane's part of a row, on its way; what does not exist is not looked at
  template <typename T>
  struct Part {
    Eight<T> a, b;
  };
  template <typename T>
  __device__ __forceinline__ void load(const T* row, Part<T>& part) const {
    if (has_a) part.a.load(row + a);
    if (has_b) part.b.load(row + b);
  }
  template <typename T>
  __device__ __forceinline__ void take(const Part<T>& part, float (&x)[16]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = has_a ? part.a[e] : 0.0f;
      x[8 + e] = has_b ? part.b[e] : 0.0f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&x)[16]) const {
    Part<T> part;
    load(row, part);
    take(part, x);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&x)[16]) const {
    if (has_a) store8(row + a, x, 0);
    if (has_b) store8(row + b, x, 8);
  }
};

// Cosines and sines of the pairs of a workgroup's tokens, [token][pair] (64 / LPR tokens of at most 8 LPR pairs).
struct Angles {
  float cos[512], sin[512];
  __device__ __forceinline__ void fill(const RotateParams& p, uint32_t token0, uint32_t tokens, bool back) {
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < tokens * p.pairs; i += 64 * kWaves) {
      const uint32_t t = i / p.pairs, j = i - t * p.pairs, token = min(token0 + t, p.tokens - 1), batch = token / p.n, at = token - batch * p.n;
      const uint32_t axis = p.axis_of ? min((uint32_t)max(p.axis_of[j], 0), p.axes - 1) : 0;
      const int position = p.positions[(int64_t)axis * p.position_axis + (int64_t)batch * p.position_b + at];
      // turns in 64 bits: the remainder to the nearest whole turn, in f32, is off by at most 2^-26 of a turn
      const double turns = (double)position * ((double)p.frequencies[j] * 0.15915494309189533577);
      float sine, cosine;
      sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &sine, &cosine);
      cos[i] = cosine;
      sin[i] = back ? -sine : sine;
    }
  }
};

// ... of a lane's columns for one token.
template <int KIND, int LPR>
struct Turn {
  static constexpr int N = KIND == kApart ? 16 : 8;
  float cos[N], sin[N];
  int count;  // halves, neighbours: pairs of this lane that turn (0 or 8; neighbours: any)

  // pair of the lane's n-th angle
  static __device__ __forceinline__ uint32_t pair(const RotateParams& p, const Columns<KIND>& c, int n) {
    const uint32_t column = c.a + n;
    if constexpr (KIND == kApart) return column < p.pairs ? column : column - p.pairs;
    if constexpr (KIND == kNeighbours) return c.a / 2 + n;
    return column;
  }
  // `token`: of the workgroup's
  __device__ __forceinline__ void set(const RotateParams& p, const Columns<KIND>& c, const Angles& angles, uint32_t token) {
    if constexpr (KIND == kHalves) count = c.b == c.a + p.pairs && c.a < p.pairs ? 8 : 0;
    else if constexpr (KIND == kNeighbours) count = min(max((int)p.pairs - (int)(c.a / 2), 0), 8);
    else count = 0;
    if (p.pairs == 0) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t at = token * p.pairs + min(pair(p, c, n), p.pairs - 1);
      cos[n] = angles.cos[at];
      sin[n] = angles.sin[at];
    }
  }
  // `mine`: LDS of this lane's row, 16 LPR + 4 floats
  __device__ __forceinline__ void turn(const RotateParams& p, const Columns<KIND>& c, float (&x)[16], float* mine) const {
    if constexpr (KIND == kApart) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int e = 0; e < 16; e += 4) *reinterpret_cast<f32x4*>(mine + c.a + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
      // (lanes of one wavefront: a wait is enough)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t column = c.a + e;
        if (column >= 2 * p.pairs) continue;
        const bool second = column >= p.pairs;
        const float other = mine[second ? column - p.pairs : column + p.pairs];
        x[e] = second ? __builtin_fmaf(other, sin[e], x[e] * cos[e]) : __builtin_fmaf(-other, sin[e], x[e] * cos[e]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
      if (count == 0) return;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int i = KIND == kHalves ? n : 2 * n, j = KIND == kHalves ? 8 + n : 2 * n + 1;
        const float u = x[i], v = x[j];
        const float first = __builtin_fmaf(-v, sin[n], u * cos[n]), second = __builtin_fmaf(u, sin[n], v * cos[n]);
        // (a column that does not turn is left as it is, whatever its neighbour holds)
        x[i] = KIND == kHalves || n < count ? first : u;
        x[j] = KIND == kHalves || n < count ? second : v;
      }
    }
  }
};

template <typename T, int KIND>
__device__ __forceinline__ void load_weight(const RotateParams& p, const Columns<KIND>& c, const void* weight, float (&w)[16]) {
  if (p.f32_weights) c.load((const float*)weight, w);
  else c.load((const T*)weight, w);
}

// A workgroup's run of heads (of queries or of keys) and the lanes' place in it.
template <int LPR>
struct Place {
  static constexpr uint32_t TOKENS = 64 / LPR;
  const RotateSide* side;
  uint32_t step, chunk_of_side, head0, head1, lane, group, wave;
  __device__ __forceinline__ explicit Place(const RotateParams& p) {
    const uint32_t chunks = p.side[0].chunks + p.side[1].chunks;
    step = blockIdx.x / chunks;
    const uint32_t chunk = blockIdx.x - step * chunks;
    const bool keys = chunk >= p.side[0].chunks;
    side = &p.side[keys];
    chunk_of_side = keys ? chunk - p.side[0].chunks : chunk;
    lane = threadIdx.x % LPR;
    group = threadIdx.x % 64 / LPR;
    wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
    head0 = chunk_of_side * p.each + wave;
    head1 = min(chunk_of_side * p.each + p.each, side->heads);
  }
  // the token of these lanes in a tile; a token past the end: the last one, and false
  __device__ __forceinline__ bool token(const RotateParams& p, uint32_t tile, uint32_t& batch, uint32_t& at) const {
    const uint32_t t = tile * TOKENS + group, inside = min(t, p.tokens - 1);
    batch = inside / p.n;
    at = inside - batch * p.n;
    return t < p.tokens;
  }
};
template <typename T>
__device__ __forceinline__ T* row_of(const RotateOperand& x, uint32_t batch, uint32_t head, uint32_t at) {
  return (T*)x.data + (int64_t)batch * x.sb + (int64_t)head * x.sh + (int64_t)at * x.sn;
}

template <typename T, int LPR, int KIND>
__device__ __forceinline__ void forward_body(const RotateParams& p) {
  __shared__ __attribute__((aligned(16))) float exchange[KIND == kApart ? kWaves * 64 / LPR : 1][KIND == kApart ? 16 * LPR + 4 : 4];
  __shared__ Angles angles;
  const Place<LPR> place(p);
  const RotateSide& side = *place.side;
  const Columns<KIND> columns(p, place.lane);
  float* const mine = exchange[KIND == kApart ? threadIdx.x / LPR : 0];
  float w[16];
  if (side.weight) load_weight<T>(p, columns, side.weight, w);
  for (uint32_t tile = place.step; tile < p.tiles; tile += p.steps) {
    uint32_t batch, at;
    const bool there = place.token(p, tile, batch, at);
    if (tile != place.step) __syncthreads();  // (those of the tile before are read)
    angles.fill(p, tile * Place<LPR>::TOKENS, Place<LPR>::TOKENS, false);
    __syncthreads();
    Turn<KIND, LPR> turn;
    turn.set(p, columns, angles, place.group);
    typename Columns<KIND>::template Part<T> next;
    if (place.head0 < place.head1) columns.load(row_of<const T>(side.x, batch, place.head0, at), next);
    for (uint32_t head = place.head0; head < place.head1; head += kWaves) {
      float x[16];
      columns.take(next, x);
      if (head + kWaves < place.head1) columns.load(row_of<const T>(side.x, batch, head + kWaves, at), next);
      if (side.weight) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum = __builtin_fmaf(x[e], x[e], sum);
        const float inverse = 1.0f / sqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), p.inverse_d, p.eps));
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = x[e] * inverse * w[e];
      }
      turn.turn(p, columns, x, mine);
      if (there) columns.store(row_of<T>(side.y, batch, head, at), x);
    }
  }
}

template <typename T, int LPR, int KIND>
__device__ __forceinline__ void backward_body(const RotateParams& p) {
  __shared__ __attribute__((aligned(16))) float exchange[KIND == kApart ? kWaves * 64 / LPR : 1][KIND == kApart ? 16 * LPR + 4 : 4];
  __shared__ float sums[kWaves][16 * LPR];
  __shared__ Angles angles;
  const Place<LPR> place(p);
  const RotateSide& side = *place.side;
  const Columns<KIND> columns(p, place.lane);
  float* const mine = exchange[KIND == kApart ? threadIdx.x / LPR : 0];
  float w[16], dw[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.0f;
  if (side.weight) load_weight<T>(p, columns, side.weight, w);
  for (uint32_t tile = place.step; tile < p.tiles; tile += p.steps) {
    uint32_t batch, at;
    const bool there = place.token(p, tile, batch, at);
    if (tile != place.step) __syncthreads();  // (those of the tile before are read)
    angles.fill(p, tile * Place<LPR>::TOKENS, Place<LPR>::TOKENS, true);
    __syncthreads();
    Turn<KIND, LPR> turn;
    turn.set(p, columns, angles, place.group);
    typename Columns<KIND>::template Part<T> next, next_x;
    auto request = [&](uint32_t head) {
      columns.load(row_of<const T>(side.g, batch, head, at), next);
      if (side.weight) columns.load(row_of<const T>(side.x, batch, head, at), next_x);
    };
    if (place.head0 < place.head1) request(place.head0);
    for (uint32_t head = place.head0; head < place.head1; head += kWaves) {
      float g[16], x[16];
      columns.take(next, g);
      if (side.weight) columns.take(next_x, x);
      if (head + kWaves < place.head1) request(head + kWaves);
      if (side.weight) {
        turn.turn(p, columns, g, mine);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum = __builtin_fmaf(x[e], x[e], sum);
        const float inverse = 1.0f / sqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), p.inverse_d, p.eps));
        float along = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] *= inverse;
          dw[e] = there ? __builtin_fmaf(g[e], x[e], dw[e]) : dw[e];
          g[e] *= w[e];
          along = __builtin_fmaf(g[e], x[e], along);
        }
        along = lanes_sum<LPR>(along) * p.inverse_d;
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e] = (g[e] - x[e] * along) * inverse;
      } else {
        turn.turn(p, columns, g, mine);
      }
      if (there) columns.store(row_of<T>(side.y, batch, head, at), g);
    }
  }
  if (!side.weight) return;
  // the wavefront's groups, then the wavefronts, in a fixed order
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int bit = LPR; bit < 64; bit <<= 1) dw[e] += __shfl_xor(dw[e], bit);
    const uint32_t column = (e < 8 ? columns.a : columns.b) + e % 8;
    if (place.group == 0 && (e < 8 ? columns.has_a : columns.has_b)) sums[place.wave][column] = dw[e];
  }
  __syncthreads();
  const uint32_t column = threadIdx.x;
  if (column >= p.d) return;
  float sum = 0.0f;
#pragma unroll
  for (int wave = 0; wave < kWaves; ++wave) sum += sums[wave][column];
  side.partial[((size_t)place.step * side.chunks + place.chunk_of_side) * p.d + column] = sum;
}

// The workgroups' shares of the weights' gradients added up: 32 columns of one weight a workgroup, 32 runs of shares.
template <typename T>
__device__ __forceinline__ void join_body(const RotateParams& p) {
  __shared__ float sums[32][33];
  const RotateSide& side = p.side[blockIdx.y];
  if (!side.weight) return;
  const uint32_t column = blockIdx.x * 32 + threadIdx.x % 32, run = threadIdx.x / 32, rows = p.steps * side.chunks;
  float sum = 0.0f;
  if (column < p.d) {
#pragma unroll 4
    for (uint32_t row = run; row < rows; row += 32) sum += side.partial[(size_t)row * p.d + column];
  }
  sums[run][threadIdx.x % 32] = sum;
  __syncthreads();
  if (run != 0 || column >= p.d) return;
#pragma unroll
  for (int r = 1; r < 32; ++r) sum += sums[r][threadIdx.x % 32];
  if (p.f32_weights) ((float*)side.weight_grad)[column] = sum;
  else ((T*)side.weight_grad)[column] = (T)sum;
}

}  // namespace rotate
