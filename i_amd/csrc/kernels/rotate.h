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
//   quads       (j, j + pairs), pairs another multiple of 4 (whole rows of 40, 72, 104 columns): the same in runs of four, of which the last
//               lane of pairs may have one less
//   neighbours  (2 j, 2 j + 1): 16 columns in a row
//   apart       (j, j + pairs) with any other number of pairs: 16 columns in a row, partners through LDS (7 sequences of 5327 tokens, 20 heads
//               of 40 columns, forward and backward: 118 us, as quads 76)
#pragma once
#include "common.h"
#include "rotate_params.h"

namespace rotate {

constexpr int kWaves = 4;
enum Kind { kHalves, kQuads, kNeighbours, kApart };

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

// N elements as they lie in memory, and as f32: 8, or 4
template <typename T, int N>
struct Run {
  static constexpr int BYTES = N * (int)sizeof(T);
  uint32_t words[BYTES / 4];
  __device__ __forceinline__ void load(const T* at) {
    if constexpr (BYTES == 8) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(at);
      words[0] = x[0];
      words[1] = x[1];
    } else {
#pragma unroll
      for (int n = 0; n < BYTES / 16; ++n) {
        const u32x4 x = ldg128(reinterpret_cast<const char*>(at) + 16 * n);
#pragma unroll
        for (int e = 0; e < 4; ++e) words[4 * n + e] = x[e];
      }
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, words[e]);
    return __builtin_bit_cast(float, e & 1 ? words[e / 2] & 0xffff0000u : words[e / 2] << 16);
  }
};
template <int N>
__device__ __forceinline__ void store_run(float* at, const float* x) {
#pragma unroll
  for (int n = 0; n < N; n += 4) *reinterpret_cast<f32x4*>(at + n) = f32x4{x[n], x[n + 1], x[n + 2], x[n + 3]};
}
template <int N>
__device__ __forceinline__ void store_run(bf16_t* at, const float* x) {
  typedef __attribute__((ext_vector_type(N))) __bf16 run_t;
  run_t v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (bf16_t)x[e];
  *reinterpret_cast<run_t*>(at) = v;
}

// The columns of a lane: two runs of 8 (quads: four of 4), those that exist.  halves, quads: the second half of the runs holds the partners
// of the first.
template <int KIND>
struct Columns {
  static constexpr int RUNS = KIND == kQuads ? 4 : 2, EACH = 16 / RUNS;
  uint32_t at[RUNS];
  bool has[RUNS];
  bool halves;  // of a pair
  __device__ __forceinline__ Columns(const RotateParams& p, uint32_t lane) {
    const uint32_t turning = KIND == kHalves || KIND == kQuads ? (p.pairs + 7) / 8 : 0;  // lanes that have pairs' halves
    halves = lane < turning;
#pragma unroll
    for (int n = 0; n < RUNS; ++n) {
      const uint32_t half = n / (RUNS / 2), of_half = 8 * lane + EACH * (n % (RUNS / 2)), rest = 2 * (KIND == kHalves || KIND == kQuads ? p.pairs : 0) + 16 * (lane - turning) + EACH * n;
      at[n] = halves ? of_half + half * p.pairs : rest;
      has[n] = halves ? of_half < p.pairs : rest < p.d;
    }
  }
  __device__ __forceinline__ uint32_t column(int e) const { return at[e / EACH] + e % EACH; }
  __device__ __forceinline__ bool exists(int e) const { return has[e / EACH]; }
  // a lane's part of a row, on its way; what does not exist is not looked at and stays zero
  template <typename T>
  struct Part {
    Run<T, EACH> run[RUNS] = {};
  };
  template <typename T>
  __device__ __forceinline__ void load(const T* row, Part<T>& part) const {
#pragma unroll
    for (int n = 0; n < RUNS; ++n)
      if (has[n]) part.run[n].load(row + at[n]);
  }
  template <typename T>
  __device__ __forceinline__ void take(const Part<T>& part, float (&x)[16]) const {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = part.run[e / EACH][e % EACH];
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&x)[16]) const {
    Part<T> part;
    load(row, part);
    take(part, x);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&x)[16]) const {
#pragma unroll
    for (int n = 0; n < RUNS; ++n)
      if (has[n]) store_run<EACH>(row + at[n], x + EACH * n);
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
      // turns in 64 bits, off by at most 3 2^-53 of them: the remainder to the nearest whole turn, in f32, is off by 2^-26 of a turn more
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
  int count;  // halves, quads, neighbours: pairs of this lane that turn (0 or 8; neighbours: any)

  // `token`: of the workgroup's
  __device__ __forceinline__ void set(const RotateParams& p, const Columns<KIND>& c, const Angles& angles, uint32_t lane, uint32_t token) {
    count = KIND == kNeighbours ? min(max((int)p.pairs - (int)(8 * lane), 0), 8) : KIND != kApart && c.halves ? 8 : 0;
    if (p.pairs == 0) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      // pair of the lane's n-th angle: (apart) that of column n;  else 8 lane + n, also where it does not turn (one of another token, or
      // anything: there are 8 LPR pairs' room), which quads multiply with a column of zero
      uint32_t pair = 8 * lane + n;
      if constexpr (KIND == kApart) {
        pair = c.at[0] + n;
        pair = min(pair < p.pairs ? pair : pair - p.pairs, p.pairs - 1);
      }
      if constexpr (KIND == kQuads) pair = min(pair, p.pairs - 1);
      cos[n] = angles.cos[token * p.pairs + pair];
      sin[n] = angles.sin[token * p.pairs + pair];
    }
  }
  // `mine`: LDS of this lane's row, 16 LPR + 4 floats
  __device__ __forceinline__ void turn(const RotateParams& p, const Columns<KIND>& c, float (&x)[16], float* mine) const {
    if constexpr (KIND == kApart) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int e = 0; e < 16; e += 4) *reinterpret_cast<f32x4*>(mine + c.at[0] + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
      // (lanes of one wavefront: a wait is enough)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t column = c.at[0] + e;
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
        const int i = KIND == kNeighbours ? 2 * n : n, j = KIND == kNeighbours ? 2 * n + 1 : 8 + n;
        const float u = x[i], v = x[j];
        const float first = __builtin_fmaf(-v, sin[n], u * cos[n]), second = __builtin_fmaf(u, sin[n], v * cos[n]);
        // (a column that does not turn is left as it is, whatever its neighbour holds)
        x[i] = KIND != kNeighbours || n < count ? first : u;
        x[j] = KIND != kNeighbours || n < count ? second : v;
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

// (With a norm and without are code of their own: decided at every row, the gradient took 192 registers instead of 152 and a compute unit
// held two workgroups instead of three: 2 x 4096 tokens of 32 and 8 heads of 128 columns 47.5 -> 38 us.)
template <typename T, int LPR, int KIND, bool NORM>
__device__ __forceinline__ void forward_rows(const RotateParams& p, const Place<LPR>& place, Angles& angles, float* mine) {
  const RotateSide& side = *place.side;
  const Columns<KIND> columns(p, place.lane);
  float w[16];
  if constexpr (NORM) load_weight<T>(p, columns, side.weight, w);
  typename Columns<KIND>::template Part<T> next;
  for (uint32_t tile = place.step; tile < p.tiles; tile += p.steps) {
    uint32_t batch, at;
    const bool there = place.token(p, tile, batch, at);
    if (tile != place.step) __syncthreads();  // (those of the tile before are read)
    angles.fill(p, tile * Place<LPR>::TOKENS, Place<LPR>::TOKENS, false);
    __syncthreads();
    Turn<KIND, LPR> turn;
    turn.set(p, columns, angles, place.lane, place.group);
    if (place.head0 < place.head1) columns.load(row_of<const T>(side.x, batch, place.head0, at), next);
    for (uint32_t head = place.head0; head < place.head1; head += kWaves) {
      float x[16];
      columns.take(next, x);
      if (head + kWaves < place.head1) columns.load(row_of<const T>(side.x, batch, head + kWaves, at), next);
      if constexpr (NORM) {
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
__device__ __forceinline__ void forward_body(const RotateParams& p) {
  __shared__ __attribute__((aligned(16))) float exchange[KIND == kApart ? kWaves * 64 / LPR : 1][KIND == kApart ? 16 * LPR + 4 : 4];
  __shared__ Angles angles;
  const Place<LPR> place(p);
  float* const mine = exchange[KIND == kApart ? threadIdx.x / LPR : 0];
  if (place.side->weight) forward_rows<T, LPR, KIND, true>(p, place, angles, mine);
  else forward_rows<T, LPR, KIND, false>(p, place, angles, mine);
}

template <typename T, int LPR, int KIND, bool NORM>
__device__ __forceinline__ void backward_rows(const RotateParams& p, const Place<LPR>& place, Angles& angles, float* mine, float (&sums)[kWaves][16 * LPR]) {
  const RotateSide& side = *place.side;
  const Columns<KIND> columns(p, place.lane);
  float w[16], dw[16];
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < 16; ++e) dw[e] = 0.0f;
    load_weight<T>(p, columns, side.weight, w);
  }
  typename Columns<KIND>::template Part<T> next, next_x;
  for (uint32_t tile = place.step; tile < p.tiles; tile += p.steps) {
    uint32_t batch, at;
    const bool there = place.token(p, tile, batch, at);
    if (tile != place.step) __syncthreads();  // (those of the tile before are read)
    angles.fill(p, tile * Place<LPR>::TOKENS, Place<LPR>::TOKENS, true);
    __syncthreads();
    Turn<KIND, LPR> turn;
    turn.set(p, columns, angles, place.lane, place.group);
    auto request = [&](uint32_t head) {
      columns.load(row_of<const T>(side.g, batch, head, at), next);
      if constexpr (NORM) columns.load(row_of<const T>(side.x, batch, head, at), next_x);
    };
    if (place.head0 < place.head1) request(place.head0);
    for (uint32_t head = place.head0; head < place.head1; head += kWaves) {
      float g[16], x[16];
      columns.take(next, g);
      if constexpr (NORM) columns.take(next_x, x);
      if (head + kWaves < place.head1) request(head + kWaves);
      turn.turn(p, columns, g, mine);
      if constexpr (NORM) {
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
      }
      if (there) columns.store(row_of<T>(side.y, batch, head, at), g);
    }
  }
  if constexpr (NORM) {
    // the wavefront's groups, then the wavefronts, in a fixed order
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
      for (int bit = LPR; bit < 64; bit <<= 1) dw[e] += __shfl_xor(dw[e], bit);
      if (place.group == 0 && columns.exists(e)) sums[place.wave][columns.column(e)] = dw[e];
    }
    __syncthreads();
    const uint32_t column = threadIdx.x;
    if (column >= p.d) return;
    float sum = 0.0f;
#pragma unroll
    for (int wave = 0; wave < kWaves; ++wave) sum += sums[wave][column];
    side.partial[((size_t)place.step * side.chunks + place.chunk_of_side) * p.d + column] = sum;
  }
}

template <typename T, int LPR, int KIND>
__device__ __forceinline__ void backward_body(const RotateParams& p) {
  __shared__ __attribute__((aligned(16))) float exchange[KIND == kApart ? kWaves * 64 / LPR : 1][KIND == kApart ? 16 * LPR + 4 : 4];
  __shared__ float sums[kWaves][16 * LPR];
  __shared__ Angles angles;
  const Place<LPR> place(p);
  float* const mine = exchange[KIND == kApart ? threadIdx.x / LPR : 0];
  if (place.side->weight) backward_rows<T, LPR, KIND, true>(p, place, angles, mine, sums);
  else backward_rows<T, LPR, KIND, false>(p, place, angles, mine, sums);
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
