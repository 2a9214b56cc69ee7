// The gradient of attention with masks, capped scores and a bias by distance, and the weight that each key received.
//
//   p = exp(s - lse)   dv_j = sum_i p_ij do_i   ds_ij = p_ij (do_i.v_j - delta_i) (1 - (x_ij / cap)^2)   delta_i = do_i.o_i
//   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i   (x: the capped score before its bias)
//   w_j = sum_i p_ij
//
// Two kernels compute the scores once each, one walking the keys of a tile of queries (dq), one the queries of a tile of keys (dk,
// dv, over all the query heads that share the key head): seven products instead of the five that atomic additions to dq would
// leave, and every sum in an order that does not change from run to run.
//
// Measured, call after call, 2 x 16 heads of 4096 x 128 bf16, all keys: dq 445 .. 453 us, dk and dv 746 us, weights 164 us (838 TFLOP/s); 1 x
// 16 heads of 2048 x 128 f32: 423, 663, 139 us.  dq is bound as the forward kernel is; of dk and dv's time see below.
#pragma once
#include "attend.h"

namespace attend {

// Query tiles of `rows` rows (a divisor of 64).
struct QueryTiles {
  const AttendParams& p;
  uint32_t batch, rows;
  __device__ __forceinline__ uint32_t count() const { return (p.nq + rows - 1) / rows; }
  __device__ __forceinline__ const char* record(uint32_t tile) const {
    return p.spans + ((size_t)batch * ((p.nq + 63) / 64) + tile * rows / 64) * kSpanRecord;
  }
  // without first and last
  __device__ __forceinline__ Spans computed(uint32_t tile) const {
    if (!p.causal) return Spans{0, 0, (int)p.nk, (int)p.nk};
    const int row0 = (int)(tile * rows), row1 = min(row0 + (int)rows, (int)p.nq) - 1;
    const int least = min(max(row0 + p.shift + 1, 0), (int)p.nk), most = min(max(row1 + p.shift + 1, 0), (int)p.nk);
    return Spans{0, 0, least, most};
  }
};

// The plan of the work on keys of a sequence, by a workgroup of 256: the query tiles first .. last that see any key of a key tile.  The
// bounds are taken from first and last themselves, 256 blocks of 64 queries at a time, so that this needs no launch of its own.
__device__ __forceinline__ void plan_sequence(const AttendParams& p, uint32_t batch) {
  constexpr uint32_t THREADS = 256, BLOCKS = 256;
  __shared__ Spans block_spans[BLOCKS];
  __shared__ int sums[THREADS / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, blocks = (p.nq + 63) / 64;
  const QueryTiles queries{p, batch, p.query_rows};
  const uint32_t query_tiles = queries.count(), per_block = 64 / p.query_rows;
  int* begin_of = p.plan + (size_t)batch * (2 * p.tiles + 1);
  int* before = begin_of + p.tiles;
  int base = 0;
  for (uint32_t t0 = 0; t0 < p.tiles; t0 += THREADS) {
    const uint32_t t = t0 + tid;
    const int k0 = (int)(t * p.tile_keys), k1 = min(k0 + (int)p.tile_keys, (int)p.nk);
    uint32_t begin = 0, end = t < p.tiles ? query_tiles : 0;
    if (p.spans) {
      begin = 0xffffffff;
      end = 0;
      for (uint32_t q0 = 0; q0 < blocks; q0 += BLOCKS) {
        const uint32_t here = min(blocks - q0, BLOCKS);
        __syncthreads();
        for (uint32_t q = wave; q < here; q += THREADS / 64) {
          Spans s;
          s.none();
          s.add(span_of(p, batch, min((q0 + q) * 64 + lane, p.nq - 1)));
          s.over_lanes<64>();
          if (lane == 0) block_spans[q] = s;
        }
        __syncthreads();
        if (t < p.tiles) {
          for (uint32_t q = 0; q < here; ++q)
            if (block_spans[q].touches(k0, k1)) {
              begin = min(begin, (q0 + q) * per_block);
              end = min((q0 + q + 1) * per_block, query_tiles);
            }
        }
      }
      begin = min(begin, end);
    } else if (p.causal && t < p.tiles) {
      begin = min((uint32_t)max(k0 - p.shift, 0) / p.query_rows, query_tiles);
    }
    const int mine = (int)((end - begin) * p.group);
    int upto = mine;
#pragma unroll
    for (int bit = 1; bit < 64; bit <<= 1) {
      const int other = __shfl_up(upto, bit);
      if ((int)lane >= bit) upto += other;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int all = 0;
    for (uint32_t w = 0; w < THREADS / 64; ++w) {
      if (w < wave) upto += sums[w];
      all += sums[w];
    }
    if (t < p.tiles) {
      begin_of[t] = (int)begin;
      before[t] = base + upto - mine;
    }
    base += all;
  }
  if (tid == 0) before[p.tiles] = base;
}
// delta of a row of few keys, by 16 lanes (lane n of them has columns 8 n .. of every 128): sum p do.v over what it sees.  do.o is the same but for
// the rounding of o to bf16, which where a few keys share the weight costs the gradients more than their own rounding (2 keys:
// dq and dk 2.8 times as far from 64 bits as rounded ones, 16: 1.3 .. 1.6, 64: 1.1; with this 1.0 up to 16 keys).  16 keys at most, since a
// lane group looks at them four at a time (documents, 2 x 16 heads of 2048: 183.9 -> 186.7 us forward and backward).  Rows of more keys whose weight is
// on one all the same keep that error (scores of deviation 3: 1.8, of 8: 3.4): for them it would take a walk over all keys.
constexpr int kFewKeys = 16;
typedef __attribute__((ext_vector_type(2))) bf16_t bf16x2;
__device__ __forceinline__ float dot8(bf16x8 a, bf16x8 b, float sum) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[e], a[e + 1]}, bf16x2{b[e], b[e + 1]}, sum, false);
  return sum;
}
__device__ __forceinline__ float dot8(f32x8 a, f32x8 b, float sum) {
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(a[e], b[e], sum);
  return sum;
}
template <typename T>
__device__ __forceinline__ float delta_of_few(const AttendParams& p, const Bend& bend, uint32_t batch, uint32_t hq, uint32_t i, Span span, float lse, int lane) {
  const uint32_t hkv = hq / p.group;
  const T* q = (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh + i * p.q.sn;
  const T* go = (const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh + i * p.grad_o.sn;
  const T* K = (const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh + span.first * p.k.sn;
  const T* V = (const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh + span.first * p.v.sn;
  const float slope2 = p.slopes ? p.slopes[hq] * Bend::I_LOG2_E : 0.0f;
  constexpr int EACH = 4;  // keys at a time: as many loads under way
  float delta = 0.0f;
  for (int j0 = span.first; j0 < span.last; j0 += EACH) {
    float s[EACH], dp[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) s[n] = dp[n] = 0.0f;
#pragma unroll 1
    for (uint32_t c = 8 * lane; c < p.d; c += 128) {
      const Frag<T> a = load_frag<T>(q + c), b = load_frag<T>(go + c);
#pragma unroll
      for (int n = 0; n < EACH; ++n) {
        const uint32_t j = min(j0 + n, span.last - 1) - span.first;  // (16 rows of 32 MiB at most)
        const Frag<T> x = load_frag<T>(K + j * (uint32_t)p.k.sn + c), y = load_frag<T>(V + j * (uint32_t)p.v.sn + c);
        s[n] = dot8(a, x, s[n]);
        dp[n] = dot8(b, y, dp[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const float away = fabsf((float)((int)i + p.shift - (j0 + n)));
      const float weight = fast_exp2(__builtin_fmaf(-slope2, away, bend.one(row_sum(s[n]))) - lse);
      if (j0 + n < span.last) delta = __builtin_fmaf(weight, row_sum(dp[n]), delta);
    }
  }
  return delta;
}
// What the other kernels need to know of every query, in blocks of 64 so that a block is one transfer; the rows past the end weigh
// nothing (lse +inf), like those that see nothing.
//   rows[b, hq, block, 64]   GRAD: lse (base 2), delta;  else lse (base 2) in two parts, hi and 2^-lo
//   spans[b, block]          first and last of the 64 queries (causal included), then their Spans
// The first p.b workgroups make the plans, the next `row_blocks` take 16 rows each, 16 lanes a row (GRAD) or 256 rows, the others a
// block of spans a wavefront.
template <typename T, bool GRAD>
__device__ __forceinline__ void prepare_body(const AttendParams& p) {
  const uint32_t tid = threadIdx.x, blocks = (p.nq + 63) / 64, per = GRAD ? 16 : 256;
  const uint64_t rows = (uint64_t)p.b * p.hq * blocks * 64;
  const uint32_t row_blocks = (uint32_t)((rows + per - 1) / per);
  if (blockIdx.x < p.b) return plan_sequence(p, blockIdx.x);
  const uint32_t id = blockIdx.x - p.b;
  if (id < row_blocks) {
    uint64_t at = (uint64_t)id * per + tid;
    if constexpr (GRAD) {
      // the first rows of all heads first: those of a causal mask see few keys and take longer
      const uint32_t bh = id % (p.b * p.hq);
      at = (uint64_t)bh * blocks * 64 + (uint64_t)(id / (p.b * p.hq)) * per + tid / 16;
    }
    if (at >= rows) return;
    const uint32_t bh = (uint32_t)(at / (blocks * 64)), i = (uint32_t)(at - (uint64_t)bh * blocks * 64), batch = bh / p.hq, hq = bh - batch * p.hq;
    const bool inside = i < p.nq;
    const float lse = inside ? p.lse[(size_t)bh * p.nq + i] : -INFINITY;
    // the factor that the kernels' scores carry, so that what it is off by its exact value is off for both
    const Bend bend(p.scale, p.cap, p.slopes != nullptr);
    const double exact = (double)lse * (bend.bent ? 1.4426950408889634 : (double)bend.mult / (double)p.scale);
    const float hi = (float)exact;
    float first = lse == -INFINITY ? INFINITY : hi, second = 0.0f;
    if constexpr (GRAD) {
      const Span span = inside ? span_of(p, batch, i) : Span{0, 0};
      const bool few = sizeof(T) == 2 && span.last - span.first <= kFewKeys;  // (o of 32 bits is good enough)
      if (inside && few) {
        second = delta_of_few<T>(p, bend, batch, hq, i, span, first, tid & 15);
      } else if (inside) {
        const T* o = (const T*)p.o.data + batch * p.o.sb + hq * p.o.sh + i * p.o.sn;
        const T* go = (const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh + i * p.grad_o.sn;
        for (uint32_t c = 8 * (tid & 15); c < p.d; c += 128) {
          const Frag<T> a = load_frag<T>(o + c), b = load_frag<T>(go + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) second = __builtin_fmaf((float)a[e], (float)b[e], second);
        }
      }
      const float all = row_sum(second);
      if (!few) second = all;
    } else {
      second = lse == -INFINITY ? 0.0f : 1.0f - 0.69314718056f * (float)(exact - (double)hi);
    }
    if (!GRAD || (tid & 15) == 0) *reinterpret_cast<float2*>(p.rows + 2 * at) = float2{first, second};
  } else if (p.spans) {
    const uint32_t block = (id - row_blocks) * 4 + tid / 64;
    if (block >= p.b * blocks) return;
    const uint32_t batch = block / blocks, row = (block - batch * blocks) * 64 + (tid & 63);
    const Span mine = span_of(p, batch, min(row, p.nq - 1));
    Spans s;
    s.none();
    s.add(mine);
    s.over_lanes<64>();
    char* record = p.spans + (size_t)block * kSpanRecord;
    *reinterpret_cast<Span*>(record + 8 * (tid & 63)) = mine;
    if ((tid & 63) == 0) *reinterpret_cast<Spans*>(record + 64 * 8) = s;
  }
}

// dS as the operand of a product: bf16 in two parts, whose sum is good to 16 bits.  With one part the rounding of dS adds as much
// to the error of dq (dk) as the rounding of dq (dk) itself (1.4 times that, and 1.0 .. 1.3 with two; see delta_of_few); the second is a product more (dq takes 1.3 times as long, dk and dv 1.18).
// P stays in one part: with its rounding, which is relative to every term, the errors of o and dv are 1.2 to 1.4 times that of rounding them.
template <typename T>
struct Split {
  static constexpr int PARTS = sizeof(T) == 2 ? 2 : 1;
  Frag<T> part[PARTS];
  __device__ __forceinline__ void set(int i, float x) {
    part[0][i] = (T)x;
    if constexpr (PARTS == 2) part[1][i] = (T)(x - (float)part[0][i]);
  }
};

// A tile of 16 KB NW keys against the queries of all heads that share them.  GRAD: dk and dv (Q and dO tiles of BQ rows), else
// the keys' weights (Q tiles).  S = Q K^T with keys as columns: a lane has one key and four consecutive queries, P and dS are the
// right operands of dV^T += dO^T P and dK^T += Q^T dS as they are.  All that a tile of queries needs comes by transfers requested
// a tile ahead; a load into registers inside the loop would have to wait for them.
//
// GRAD at 128 columns holds K, V, dK and dV of 32 keys a wavefront, 320 registers: one wavefront a SIMD, whose matrix instructions, LDS reads and
// exponentials follow one another (a third of the matrix units' time); the operands in accumulation registers and reads a step
// ahead are what that leaves.  Equal runs, since key tiles see unequal numbers of queries: packed documents, 2 x 16 heads of 2048, 137 us
// with a workgroup per key tile, 68 with runs and 11 for their join.  (f32 of 256 columns fills all 512 registers and spills 80: its
// K, V, dK and dV alone are 256.)
template <typename T, int DPAD, int DUSE, int BQ, int NW, int KB, bool GRAD>
__device__ __forceinline__ void keys_body(const AttendParams& p) {
  using L = Tile<T, DPAD, BQ>;
  constexpr int BK = 16 * KB * NW, KS = DUSE / 32, DT = DUSE / 16, TILES = GRAD ? 2 : 1;
  static_assert(64 % BQ == 0 && BQ % 32 == 0 && NW >= 3, "query tile");
  __shared__ __attribute__((aligned(1024))) char smem[2][TILES][L::BYTES];  // [buffer][Q, dO]
  __shared__ __attribute__((aligned(16))) float row_of[2][BQ][2];
  __shared__ __attribute__((aligned(16))) Span span_of_row[2][BQ];
  __shared__ __attribute__((aligned(16))) Spans spans_of_tile[2];

  uint32_t head, share;
  xcd_map(blockIdx.x, p.shares, p.b * p.hkv, head, share);
  if (head >= p.b * p.hkv) return;
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const T* K = (const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh;
  const T* V = (const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh;
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<2 * TILES * L::BYTES, 64 * NW>(&smem[0][0][0], tid);

  const QueryTiles queries{p, batch, BQ};
  const int* begin_of = p.plan + (size_t)batch * (2 * p.tiles + 1);
  const int* before = begin_of + p.tiles;
  const Deal deal((uint32_t)before[p.tiles], p.shares);
  uint32_t item = share < deal.shares ? deal.begin(share) : 0;
  const uint32_t stop = share < deal.shares ? deal.begin(share + 1) : 0;

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[0][0][0]);
  const uint32_t lds_rows = lds_address(&row_of[0][0][0]), lds_spans = lds_address(&span_of_row[0][0]), lds_tile = lds_address(&spans_of_tile[0]);
  const typename L::template Requests<NW> of_q((uint32_t)(p.q.sn * sizeof(T)), p.d, wave, lane), of_g((uint32_t)(p.grad_o.sn * sizeof(T)), p.d, wave, lane);
  const uint32_t blocks = (p.nq + 63) / 64;
  auto request = [&](uint32_t hq, uint32_t t, int buf) {
    const char* Q = (const char*)((const T*)p.q.data + batch * p.q.sb + hq * p.q.sh);
    of_q(Q, (int)(t * BQ), 0, (int)p.nq, lds + buf * TILES * L::BYTES);
    if constexpr (GRAD) {
      const char* G = (const char*)((const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh);
      of_g(G, (int)(t * BQ), 0, (int)p.nq, lds + (buf * TILES + 1) * L::BYTES);
    }
    if (wave == 0) {
      const char* rows = (const char*)(p.rows + 2 * (((size_t)batch * p.hq + hq) * blocks * 64 + t * BQ));
      if (lane < BQ / 2) dma16(rows, 16 * lane, lds_rows + buf * (8 * BQ));
    }
    if (p.spans) {
      const char* record = queries.record(t);
      if (wave == 1 && lane < BQ / 2) dma16(record + t * BQ % 64 * 8, 16 * lane, lds_spans + buf * (8 * BQ));
      if (wave == 2 && lane == 0) dma16(record + 64 * 8, 0, lds_tile + buf * 16);
    }
  };

  int buf = 0;
  uint32_t slope_of = 0xffffffff;
  float slope2 = 0.0f;
  Frag<T> kf[KB][KS], vf[GRAD ? KB : 1][GRAD ? KS : 1];
  f32x4 dk[GRAD ? KB : 1][GRAD ? DT : 1], dv[GRAD ? KB : 1][GRAD ? DT : 1];
  float weight[KB];
  // keys that nobody sees, the key tiles dealt out to the shares
  const uint32_t mine0 = (uint32_t)((uint64_t)p.tiles * share / p.shares), mine1 = (uint32_t)((uint64_t)p.tiles * (share + 1) / p.shares);
  for (uint32_t t0 = mine0 + 64 * wave; t0 < mine1; t0 += 64 * NW) {
    uint64_t unseen = __builtin_amdgcn_ballot_w64(t0 + lane < mine1 && before[t0 + lane] == before[t0 + lane + 1]);
    for (; unseen; unseen &= unseen - 1) {
      const uint32_t k0 = (t0 + __builtin_ctzll(unseen)) * BK, k1 = min(k0 + BK, p.nk);
      if constexpr (GRAD) {
        for (uint32_t i = lane; i < (k1 - k0) * (p.d / 4); i += 64) {
          const uint32_t key = k0 + i / (p.d / 4), col = 4 * (i % (p.d / 4));
          store4((T*)p.grad_k.data + batch * p.grad_k.sb + hkv * p.grad_k.sh + key * p.grad_k.sn + col, f32x4{0, 0, 0, 0});
          store4((T*)p.grad_v.data + batch * p.grad_v.sb + hkv * p.grad_v.sh + key * p.grad_v.sn + col, f32x4{0, 0, 0, 0});
        }
      } else {
        for (uint32_t key = k0 + lane; key < k1; key += 64) p.weights_out[(size_t)head * p.nk + key] = p.weights_in ? p.weights_in[(size_t)head * p.nk + key] : 0.0f;
      }
    }
  }
  if (item >= stop) return;
  // the key tile of the first triple: the last one that begins at or before it, 64 looked at together
  uint32_t tile = 0;
  for (uint32_t t0 = 0; t0 < p.tiles; t0 += 64) {
    const uint64_t begun = __builtin_amdgcn_ballot_w64(t0 + lane < p.tiles && (uint32_t)before[min(t0 + lane, p.tiles)] <= item);
    if (begun == 0) break;
    tile = t0 + 63 - __builtin_clzll(begun);
    if (begun != ~0ull) break;
  }
  __syncthreads();  // (the tile memory is clear)
  while (item < stop) {
    while ((uint32_t)before[tile + 1] <= item) ++tile;
    const uint32_t tile_begin = (uint32_t)before[tile], tile_end = (uint32_t)before[tile + 1], segment_begin = item, segment_end = min(stop, tile_end);
    const uint32_t begin = (uint32_t)begin_of[tile], per = (tile_end - tile_begin) / p.group;
    const int k0 = (int)(tile * BK), kw0 = k0 + wave * (16 * KB), kw1 = min(kw0 + 16 * KB, (int)p.nk);
    auto place = [&](uint32_t n, uint32_t& hq, uint32_t& t) {
      const uint32_t h = (n - tile_begin) / per;
      hq = hkv * p.group + h;
      t = begin + (n - tile_begin - h * per);
    };
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      weight[b] = 0.0f;
      const int64_t key = min(kw0 + 16 * b + r, (int)p.nk - 1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t col = 32 * ks + 8 * g;
        kf[b][ks] = col < p.d ? load_frag<T>(K + key * p.k.sn + col) : zero_frag<T>();
        if constexpr (GRAD) vf[b][ks] = col < p.d ? load_frag<T>(V + key * p.v.sn + col) : zero_frag<T>();
      }
    }
    if constexpr (GRAD) {
      clear_sums<T>(dk);
      clear_sums<T>(dv);
    }
    uint32_t hq = 0, t = 0;
    place(item, hq, t);
    request(hq, t, buf);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      arrive(kf[b]);
      if constexpr (GRAD) {
        arrive(vf[b]);
        keep(kf[b]);
        keep(vf[b]);
      }
    }
    for (; item < segment_end; ++item, buf ^= 1) {
      const uint32_t this_t = t;
      if (p.slopes && hq != slope_of) {
        slope_of = hq;
        slope2 = p.slopes[hq] * Bend::I_LOG2_E;
        asm volatile("" : "+v"(slope2));
      }
      dma_wait_all();
      __syncthreads();
      if (item + 1 < segment_end) {
        place(item + 1, hq, t);
        request(hq, t, buf ^ 1);
      }
      Spans spans = queries.computed(this_t);
      if (p.spans) {
        spans = spans_of_tile[buf];
        spans.uniform();
      }
      // Rows of q and grad_o of queries that see nothing may hold anything: they become zeros, which P and dS of zero leave alone.
      // (The same in every wavefront.  The last one always sees a key where nothing but the causal mask hides any, so that the
      // copies of it past the end need no care.)
      if constexpr (GRAD) {
        if (spans.last_least <= 0) {
#pragma unroll 1
          for (int at = 64 * wave + lane_now(); at < L::BYTES / 16; at += 64 * NW) {
            const int row = at / L::CH;
            const bool blind = p.spans ? span_of_row[buf][row].first >= span_of_row[buf][row].last : (int)(this_t * BQ) + row + p.shift < 0;
            if (!blind) continue;
#pragma unroll
            for (int n = 0; n < TILES; ++n) *reinterpret_cast<u32x4*>(&smem[buf][n][16 * at]) = u32x4{0, 0, 0, 0};
          }
          __syncthreads();
        }
      }
      if (!spans.touches(kw0, kw1)) continue;
      const bool whole = spans.whole(kw0, kw1);
      const char* tq = &smem[buf][0][0];
      const char* tg = &smem[buf][TILES - 1][0];
      // Operands are read a step ahead of the matrix instructions that take them: with one wavefront on a SIMD nothing else
      // covers the latency of LDS.  Steps of SLABS slabs of 16 rows (row operands of Q and dO), then of COLS column blocks (transposed ones).
      constexpr int SLABS = 2, COLS = 2;
      constexpr int STEPS = (KS + SLABS - 1) / SLABS;
      Frag<T> row_q[2][SLABS], row_g[2][SLABS], col_q[2][COLS], col_g[2][COLS];
      auto fetch_rows = [&](int n) {  // step n of the tile: block n / STEPS
#pragma unroll
        for (int x = 0; x < SLABS; ++x) {
          const int ks = n % STEPS * SLABS + x;
          if (ks >= KS) continue;
          row_q[n & 1][x] = reader.rows(tq, n / STEPS, ks);
          if constexpr (GRAD) row_g[n & 1][x] = reader.rows(tg, n / STEPS, ks);
        }
      };
      auto fetch_columns = [&](int u, int step) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          col_g[step & 1][c] = reader.across(tg, step * COLS + c, u);
          col_q[step & 1][c] = reader.across(tq, step * COLS + c, u);
        }
      };
      fetch_rows(0);
#pragma unroll
      for (int u = 0; u < BQ / 32; ++u) {
        Frag<T> pf[KB];
        Split<T> df[KB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int block = 2 * u + h, row = 16 * block + 4 * g;
          f32x4 s[KB], dp[KB];
#pragma unroll
          for (int step = 0; step < STEPS; ++step) {
            const int n = block * STEPS + step;
            if (step + 1 < STEPS || h == 0 || (!GRAD && u + 1 < BQ / 32)) fetch_rows(n + 1);
            else if constexpr (GRAD) fetch_columns(u, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < SLABS; ++x) {
              const int ks = step * SLABS + x;
              if (ks >= KS) continue;
#pragma unroll
              for (int b = 0; b < KB; ++b) {
                if constexpr (GRAD) {
                  mma_kept(s[b], row_q[n & 1][x], kf[b][ks], ks == 0);
                  mma_kept(dp[b], row_g[n & 1][x], vf[b][ks], ks == 0);
                } else {
                  s[b] = mma(row_q[n & 1][x], kf[b][ks], ks == 0 ? f32x4{0, 0, 0, 0} : s[b]);
                }
              }
            }
          }
          settle<T>(s);
          if constexpr (GRAD) settle<T>(dp);
          const f32x4 pair0 = *reinterpret_cast<const f32x4*>(&row_of[buf][row][0]), pair1 = *reinterpret_cast<const f32x4*>(&row_of[buf][row + 2][0]);
          const float lse[4] = {pair0[0], pair0[2], pair1[0], pair1[2]};
          const f32x4 other = {pair0[1], pair0[3], pair1[1], pair1[3]};  // delta, or what the sum is weighed with
          if (bend.bent) bend.all(s);
          if constexpr (GRAD) {
#pragma unroll
            for (int b = 0; b < KB; ++b) dp[b] -= other;
            if (bend.capped) {
#pragma unroll
              for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) dp[b][i] *= bend.slope(s[b][i]);
            }
          }
          if (p.slopes) {
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              const float away = (float)((int)(this_t * BQ) + row + p.shift - (kw0 + 16 * b + r));
#pragma unroll
              for (int i = 0; i < 4; ++i) s[b][i] = __builtin_fmaf(-slope2, fabsf(away + (float)i), s[b][i]);
            }
          }
          if (!whole) {
            Span span[4];
            if (p.spans) {
#pragma unroll
              for (int i = 0; i < 4; ++i) span[i] = span_of_row[buf][row + i];
            } else {
              const int last = p.causal ? (int)(this_t * BQ) + row + p.shift + 1 : (int)p.nk;
#pragma unroll
              for (int i = 0; i < 4; ++i) span[i] = Span{0, p.causal ? last + i : last};
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t seen = (uint32_t)max(span[i].last - span[i].first, 0);
#pragma unroll
              for (int b = 0; b < KB; ++b)
                if ((uint32_t)(kw0 + 16 * b + r - span[i].first) >= seen) {
                  s[b][i] = -INFINITY;
                  dp[b][i] = 0.0f;
                }
            }
          }
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = fast_exp2(__builtin_fmaf(s[b][i], bend.mult, -lse[i]));
              if constexpr (GRAD) {
                pf[b][4 * h + i] = (T)e;
                df[b].set(4 * h + i, e * dp[b][i]);
              } else {
                weight[b] = __builtin_fmaf(e, other[i], weight[b]);
              }
            }
        }
        if constexpr (GRAD) {
          ready(pf);
#pragma unroll
          for (int b = 0; b < KB; ++b) ready(df[b].part);
#pragma unroll
          for (int step = 0; step < DT / COLS; ++step) {
            if (step + 1 < DT / COLS) fetch_columns(u, step + 1);
            else if (u + 1 < BQ / 32) fetch_rows((2 * u + 2) * STEPS);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
              for (int b = 0; b < KB; ++b) {
                add_mma(dv[b][step * COLS + c], col_g[step & 1][c], pf[b]);
#pragma unroll
                for (int n = 0; n < Split<T>::PARTS; ++n) add_mma(dk[b][step * COLS + c], col_q[step & 1][c], df[b].part[n]);
              }
          }
        }
      }
    }
    if constexpr (GRAD) {
      settled<T>(dk);
      settled<T>(dv);
    }

    const bool all = segment_begin == tile_begin && segment_end == tile_end;
    const size_t slot = (((size_t)head * p.shares + share) * 2 + (segment_begin == tile_begin ? 1 : 0)) * BK;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int key = kw0 + 16 * b + r;
      if constexpr (!GRAD) {
        const float sum = groups_sum(weight[b]);
        if (key >= (int)p.nk || g != 0) continue;
        const size_t to = (size_t)head * p.nk + key;
        if (!all) p.partial_k[slot + key - k0] = sum;
        else p.weights_out[to] = p.weights_in ? p.weights_in[to] + sum : sum;
      } else {
        if (key >= (int)p.nk) continue;
        T* gk = (T*)p.grad_k.data + batch * p.grad_k.sb + hkv * p.grad_k.sh + key * p.grad_k.sn;
        T* gv = (T*)p.grad_v.data + batch * p.grad_v.sb + hkv * p.grad_v.sh + key * p.grad_v.sn;
        const size_t to = (slot + key - k0) * p.d;
#pragma unroll
        for (int c = 0; c < DT; ++c)
          if (16 * c + 4 * g < p.d) {
            if (!all) {
              store4(p.partial_k + to + 16 * c + 4 * g, dk[b][c] * p.scale);
              store4(p.partial_v + to + 16 * c + 4 * g, dv[b][c]);
            } else {
              store4(gk + 16 * c + 4 * g, dk[b][c] * p.scale);
              store4(gv + 16 * c + 4 * g, dv[b][c]);
            }
          }
      }
    }
  }
}

// The shares of a key tile's result added up in their order; a workgroup per key tile of a key head.  slot(n): of the n-th share.
struct TileShares {
  uint32_t first, count;
  size_t base;
  __device__ __forceinline__ TileShares(const AttendParams& p, uint32_t head, uint32_t tile) : first(0), count(0) {
    const int* before = p.plan + (size_t)(head / p.hkv) * (2 * p.tiles + 1) + p.tiles;
    const uint32_t begin = (uint32_t)before[tile], end = (uint32_t)before[tile + 1];
    base = (size_t)head * p.shares * 2;
    if (begin == end) return;
    const Deal deal((uint32_t)before[p.tiles], p.shares);
    first = deal.of(begin);
    count = deal.of(end - 1) - first + 1;
  }
  __device__ __forceinline__ size_t slot(uint32_t n) const { return base + 2 * (first + n) + (n == 0 ? 1 : 0); }
};

template <typename T>
__device__ __forceinline__ void join_gradients_body(const AttendParams& p) {
  const uint32_t head = blockIdx.x / p.tiles, tile = blockIdx.x - head * p.tiles, batch = head / p.hkv, hkv = head - batch * p.hkv;
  const TileShares of(p, head, tile);
  if (of.count < 2) return;
  const uint32_t k0 = tile * p.tile_keys, keys = min(p.tile_keys, p.nk - k0), fours = p.d / 4;
  for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < keys * fours; i += gridDim.y * 256) {
    const uint32_t key = i / fours, col = 4 * (i - key * fours);
    f32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t n = 0; n < of.count; ++n) {
      const size_t at = (of.slot(n) * p.tile_keys + key) * p.d + col;
      k += *reinterpret_cast<const f32x4*>(p.partial_k + at);
      v += *reinterpret_cast<const f32x4*>(p.partial_v + at);
    }
    store4((T*)p.grad_k.data + batch * p.grad_k.sb + hkv * p.grad_k.sh + (k0 + key) * p.grad_k.sn + col, k);
    store4((T*)p.grad_v.data + batch * p.grad_v.sb + hkv * p.grad_v.sh + (k0 + key) * p.grad_v.sn + col, v);
  }
}

__device__ __forceinline__ void join_weights_body(const AttendParams& p) {
  const uint32_t head = blockIdx.x / p.tiles, tile = blockIdx.x - head * p.tiles, key = tile * p.tile_keys + threadIdx.x;
  const TileShares of(p, head, tile);
  if (of.count < 2 || threadIdx.x >= p.tile_keys || key >= p.nk) return;
  float sum = 0.0f;
#pragma unroll 8
  for (uint32_t n = 0; n < of.count; ++n) sum += p.partial_k[of.slot(n) * p.tile_keys + threadIdx.x];
  const size_t to = (size_t)head * p.nk + key;
  p.weights_out[to] = p.weights_in ? p.weights_in[to] + sum : sum;
}

// dq of 16 QB NW / HALVES queries: the forward kernel's walk with two products of a tile (scores, dO V^T) and dQ^T += K^T dS^T.
template <typename T, int DPAD, int DUSE, int BN, int NW, int QB, int HALVES = 1>
__device__ __forceinline__ void queries_body(const AttendParams& p) {
  using L = Tile<T, DPAD, BN>;
  constexpr int ROW_WAVES = NW / HALVES, BM = 16 * QB * ROW_WAVES, KEYS = BN / HALVES, KS = DUSE / 32, DT = DUSE / 16;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ Spans shared_spans[NW];
  __shared__ Span span_of_row[BM];

  uint32_t head, tile;
  xcd_map(blockIdx.x, p.tiles, p.b * p.hq, head, tile);
  if (head >= p.b * p.hq) return;
  if (p.causal) tile = p.tiles - 1 - tile;
  const uint32_t batch = head / p.hq, hq = head - batch * p.hq, hkv = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int half = wave / ROW_WAVES, row_wave = wave % ROW_WAVES;
  const uint32_t row0 = tile * BM + row_wave * (16 * QB);

  const T* Q = (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh;
  const T* G = (const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh;
  const char* K = (const char*)((const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh);
  const char* V = (const char*)((const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh);

  Frag<T> qf[QB][KS], gf[QB][KS];
  f32x4 dq[QB][DT];
  float lse[QB], delta[QB];
  Span span[QB];
  Spans mine;
  mine.none();
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const uint32_t row = min(row0 + 16 * b + r, p.nq - 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t col = 32 * ks + 8 * g;
      qf[b][ks] = col < p.d ? load_frag<T>(Q + row * p.q.sn + col) : zero_frag<T>();
      gf[b][ks] = col < p.d ? load_frag<T>(G + row * p.grad_o.sn + col) : zero_frag<T>();
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[b][t] = f32x4{0, 0, 0, 0};
    const float2 pair = *reinterpret_cast<const float2*>(p.rows + 2 * (((size_t)batch * p.hq + hq) * ((p.nq + 63) / 64 * 64) + row));
    lse[b] = pair.x;
    delta[b] = pair.y;
    span[b] = span_of(p, batch, row);
    mine.add(span[b]);
    if (half == 0 && g == 0) span_of_row[row_wave * (16 * QB) + 16 * b + r] = span[b];
  }
  mine.over_lanes<16>();
  mine.uniform();
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<4 * L::BYTES, 64 * NW>(&smem[0][0][0], tid);
  if (lane == 0) shared_spans[wave] = mine;
  __syncthreads();
  Spans all = shared_spans[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) all.add(shared_spans[w]);
  all.uniform();

  const float slope2 = p.slopes ? p.slopes[hq] * Bend::I_LOG2_E : 0.0f;
  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[0][0][0]);
  const int lo = all.first_least, hi = all.last_most;
  const Gap gap = p.first || p.last ? gap_between(span_of_row, BM) : Gap{0x7fffffff, 0};
  const typename L::template Requests<NW> of_k((uint32_t)(p.k.sn * sizeof(T)), p.d, wave, lane), of_v((uint32_t)(p.v.sn * sizeof(T)), p.d, wave, lane);
  auto request = [&](int k0, int buf) {
    of_k(K, k0, lo, hi, lds + (2 * buf) * L::BYTES);
    of_v(V, k0, lo, hi, lds + (2 * buf + 1) * L::BYTES);
  };
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    arrive(qf[b]);
    arrive(gf[b]);
  }
  arrive(lse);
  arrive(delta);
  if (lo < hi) {
    int k0 = lo / BN * BN, buf = 0;
    request(k0, 0);
    for (; k0 < hi; k0 += BN, buf ^= 1) {
      dma_wait_all();
      __syncthreads();
      if (k0 + BN < hi) request(k0 + BN, buf ^ 1);
      if (gap.touches(k0, k0 + BN)) {
        const uint64_t unseen = unseen_keys<BN>(span_of_row, BM, k0, lo, hi);
        if (unseen) {
          clear_rows<L, NW>(&smem[buf][0][0], unseen, wave);
          __syncthreads();
        }
      }
      const int here = k0 + half * KEYS;
      if (!mine.touches(here, here + KEYS)) continue;
      const bool whole = mine.whole(here, here + KEYS);
      const char* tk = &smem[buf][0][half * KEYS * L::RB];
      const char* tv = &smem[buf][1][half * KEYS * L::RB];
#pragma unroll
      for (int u = 0; u < KEYS / 32; ++u) {
        Split<T> df[QB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int block = 2 * u + h;
          f32x4 s[QB], dp[QB];
#pragma unroll
          for (int b = 0; b < QB; ++b) s[b] = dp[b] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const Frag<T> a = reader.rows(tk, block, ks);
#pragma unroll
            for (int b = 0; b < QB; ++b) s[b] = mma(a, qf[b][ks], s[b]);
            const Frag<T> v = reader.rows(tv, block, ks);
#pragma unroll
            for (int b = 0; b < QB; ++b) dp[b] = mma(v, gf[b][ks], dp[b]);
          }
          settle<T>(s);
          settle<T>(dp);
          if (bend.bent) bend.all(s);
#pragma unroll
          for (int b = 0; b < QB; ++b) dp[b] -= delta[b];
          if (bend.capped) {
#pragma unroll
            for (int b = 0; b < QB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) dp[b][i] *= bend.slope(s[b][i]);
          }
          if (p.slopes) {
#pragma unroll
            for (int b = 0; b < QB; ++b) {
              const float away = (float)((int)(row0 + 16 * b) + r + p.shift - here - 16 * block - 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i) s[b][i] = __builtin_fmaf(-slope2, fabsf(away - (float)i), s[b][i]);
            }
          }
          if (!whole) {
#pragma unroll
            for (int b = 0; b < QB; ++b) {
              const uint32_t seen = (uint32_t)max(span[b].last - span[b].first, 0);
              const int at = here + 16 * block + 4 * g - span[b].first;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if ((uint32_t)(at + i) >= seen) {
                  s[b][i] = -INFINITY;
                  dp[b][i] = 0.0f;
                }
            }
          }
#pragma unroll
          for (int b = 0; b < QB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) df[b].set(4 * h + i, fast_exp2(__builtin_fmaf(s[b][i], bend.mult, -lse[b])) * dp[b][i]);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const Frag<T> a = reader.across(tk, t, u);
#pragma unroll
          for (int b = 0; b < QB; ++b)
#pragma unroll
            for (int n = 0; n < Split<T>::PARTS; ++n) dq[b][t] = mma(a, df[b].part[n], dq[b][t]);
        }
      }
    }
  }
  if constexpr (HALVES == 2) {
    static_assert(ROW_WAVES * QB * DT * 1024 <= 4 * L::BYTES, "the results of a half fit the tiles");
    char* const left = &smem[0][0][0] + row_wave * (QB * DT * 1024) + 16 * lane;
    __syncthreads();
    if (half == 1) {
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(left + 1024 * (b * DT + t)) = dq[b][t];
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
      for (int t = 0; t < DT; ++t) dq[b][t] += *reinterpret_cast<const f32x4*>(left + 1024 * (b * DT + t));
  }
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const uint32_t row = row0 + 16 * b + r;
    if (row >= p.nq) continue;
    T* out = (T*)p.grad_q.data + batch * p.grad_q.sb + hq * p.grad_q.sh + row * p.grad_q.sn;
#pragma unroll
    for (int t = 0; t < DT; ++t)
      if (16 * t + 4 * g < p.d) store4(out + 16 * t + 4 * g, dq[b][t] * p.scale);
  }
}

// The same for few queries: 16 a workgroup, its NW wavefronts walking tiles of 32 keys of their own (see forward_few_body), whose
// shares of dq are added up in LDS in the wavefronts' order.
template <typename T, int DPAD, int DUSE, int NW>
__device__ __forceinline__ void queries_few_body(const AttendParams& p) {
  using L = Tile<T, DPAD, 32>;
  constexpr int KS = DUSE / 32, DT = DUSE / 16, LOADS = 2 * L::WL;
  __shared__ __attribute__((aligned(1024))) char smem[NW][2][2][L::BYTES];  // [wavefront][buffer][K, V]

  uint32_t head, tile;
  xcd_map(blockIdx.x, p.tiles, p.b * p.hq, head, tile);
  if (head >= p.b * p.hq) return;
  const uint32_t batch = head / p.hq, hq = head - batch * p.hq, hkv = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t row0 = 16 * tile, row = min(row0 + r, p.nq - 1);
  const T* Q = (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh + row * p.q.sn;
  const T* G = (const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh + row * p.grad_o.sn;
  const char* K = (const char*)((const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh);
  const char* V = (const char*)((const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh);

  Frag<T> qf[KS], gf[KS];
  f32x4 dq[DT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const uint32_t col = 32 * ks + 8 * g;
    qf[ks] = col < p.d ? load_frag<T>(Q + col) : zero_frag<T>();
    gf[ks] = col < p.d ? load_frag<T>(G + col) : zero_frag<T>();
  }
#pragma unroll
  for (int t = 0; t < DT; ++t) dq[t] = f32x4{0, 0, 0, 0};
  const float2 pair = *reinterpret_cast<const float2*>(p.rows + 2 * (((size_t)batch * p.hq + hq) * ((p.nq + 63) / 64 * 64) + row));
  float lse[1] = {pair.x}, delta[1] = {pair.y};
  const Span span = span_of(p, batch, row);
  Spans all;
  all.none();
  all.add(span);
  all.over_lanes<16>();
  all.uniform();
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<NW * 4 * L::BYTES, 64 * NW>(&smem[0][0][0][0], tid);

  const float slope2 = p.slopes ? p.slopes[hq] * Bend::I_LOG2_E : 0.0f;
  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[wave][0][0][0]);
  const int lo = all.first_least, hi = all.last_most;
  const Gap gap = p.first || p.last ? gap_between(span) : Gap{0x7fffffff, 0};
  const typename L::template Requests<1> of_k((uint32_t)(p.k.sn * sizeof(T)), p.d, 0, lane), of_v((uint32_t)(p.v.sn * sizeof(T)), p.d, 0, lane);
  auto request = [&](int k0, int buf) {
    of_k(K, k0, lo, hi, lds + (2 * buf) * L::BYTES);
    of_v(V, k0, lo, hi, lds + (2 * buf + 1) * L::BYTES);
  };
  arrive(qf);
  arrive(gf);
  arrive(lse);
  arrive(delta);
  __syncthreads();
  int k0 = lo < hi ? lo / 32 * 32 + 32 * wave : hi;
  if (k0 < hi) {
    request(k0, 0);
    for (int buf = 0; k0 < hi; k0 += 32 * NW, buf ^= 1) {
      if (k0 + 32 * NW < hi) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request(k0 + 32 * NW, buf ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS < 63 ? LOADS : 63) : "memory");
      } else {
        dma_wait_all();
      }
      const bool whole = all.whole(k0, k0 + 32);
      if (gap.touches(k0, k0 + 32)) {
        const uint64_t unseen = seen_keys(Span{lo, hi}, k0) & ~(uint64_t)row_or((uint32_t)seen_keys(span, k0)) & 0xffffffffu;
        if (unseen) clear_rows<L, 1>(&smem[wave][buf][0][0], unseen, 0);
      }
      const char* tk = &smem[wave][buf][0][0];
      const char* tv = &smem[wave][buf][1][0];
      f32x4 s[2], dp[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = dp[h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s[h] = mma(reader.rows(tk, h, ks), qf[ks], s[h]);
          dp[h] = mma(reader.rows(tv, h, ks), gf[ks], dp[h]);
        }
      }
      settle<T>(s);
      settle<T>(dp);
      if (bend.bent) bend.all(s);
      Split<T> df;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k0 + 16 * h + 4 * g;
        dp[h] -= delta[0];
        if (bend.capped) {
#pragma unroll
          for (int i = 0; i < 4; ++i) dp[h][i] *= bend.slope(s[h][i]);
        }
        if (p.slopes) {
          const float away = (float)((int)row0 + r + p.shift - at);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][i] = __builtin_fmaf(-slope2, fabsf(away - (float)i), s[h][i]);
        }
        if (!whole) {
          const uint32_t seen = (uint32_t)max(span.last - span.first, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((uint32_t)(at + i - span.first) >= seen) {
              s[h][i] = -INFINITY;
              dp[h][i] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) df.set(4 * h + i, fast_exp2(__builtin_fmaf(s[h][i], bend.mult, -lse[0])) * dp[h][i]);
      }
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const Frag<T> a = reader.across(tk, t, 0);
#pragma unroll
        for (int n = 0; n < Split<T>::PARTS; ++n) dq[t] = mma(a, df.part[n], dq[t]);
      }
    }
  }
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(&smem[wave][0][0][0]);
#pragma unroll
  for (int t = 0; t < DT; ++t) store4(mine + r * DPAD + 4 * ((4 * t + g) ^ r), dq[t]);
  __syncthreads();
  const uint32_t fours = p.d / 4, count = min(16u, p.nq - row0);
  for (uint32_t i = tid; i < count * fours; i += 64 * NW) {
    const uint32_t n = i / fours, c = i - n * fours;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(&smem[w][0][0][0]) + n * DPAD + 4 * (c ^ n));
    store4((T*)p.grad_q.data + batch * p.grad_q.sb + hq * p.grad_q.sh + (row0 + n) * p.grad_q.sn + 4 * c, sum * p.scale);
  }
}

}  // namespace attend
