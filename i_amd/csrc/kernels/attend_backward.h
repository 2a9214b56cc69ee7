// The gradient of attention with masks, capped scores and a bias by distance, and the weight that each key received.
//
//   p = exp(s - lse)   dv_j = sum_i p_ij do_i   ds_ij = p_ij (do_i.v_j - delta_i) (1 - (x_ij / cap)^2)   delta_i = do_i.o_i
//   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i   (x: the capped score before its bias)
//   w_j = sum_i p_ij
//
// Two kernels compute the scores once each, one walking the keys of a tile of queries (dq), one the queries of a tile of keys (dk,
// dv, over all the query heads that share the key head): seven products instead of the five that atomic additions to dq would
// leave, and every sum in an order that does not change from run to run.
#pragma once
#include "attend.h"

namespace attend {

// What the other kernels need to know of every query, in blocks of 64 so that a block is one transfer; the rows past the end weigh
// nothing (lse +inf), like those that see nothing.
//   rows[b, hq, block, 64]   GRAD: lse (base 2), delta;  else lse (base 2) in two parts, hi and 2^-lo
//   spans[b, block]          first and last of the 64 queries (causal included), then their Spans
// The first `row_blocks` workgroups take 16 rows each, 16 lanes a row (GRAD) or 256 rows, the others a block of spans a wavefront.
template <typename T, bool GRAD>
__device__ __forceinline__ void prepare_body(const AttendParams& p) {
  const uint32_t tid = threadIdx.x, blocks = (p.nq + 63) / 64, per = GRAD ? 16 : 256;
  const uint64_t rows = (uint64_t)p.b * p.hq * blocks * 64;
  const uint32_t row_blocks = (uint32_t)((rows + per - 1) / per);
  if (blockIdx.x < row_blocks) {
    const uint64_t at = (uint64_t)blockIdx.x * per + (GRAD ? tid / 16 : tid);
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
      if (inside) {
        const T* o = (const T*)p.o.data + batch * p.o.sb + hq * p.o.sh + i * p.o.sn;
        const T* go = (const T*)p.grad_o.data + batch * p.grad_o.sb + hq * p.grad_o.sh + i * p.grad_o.sn;
        for (uint32_t c = 8 * (tid & 15); c < p.d; c += 128) {
          const Frag<T> a = load_frag<T>(o + c), b = load_frag<T>(go + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) second = __builtin_fmaf((float)a[e], (float)b[e], second);
        }
      }
#pragma unroll
      for (int bit = 1; bit < 16; bit <<= 1) second += __shfl_xor(second, bit);
    } else {
      second = lse == -INFINITY ? 0.0f : 1.0f - 0.69314718056f * (float)(exact - (double)hi);
    }
    if (!GRAD || (tid & 15) == 0) *reinterpret_cast<float2*>(p.rows + 2 * at) = float2{first, second};
  } else if (p.spans) {
    const uint32_t block = (blockIdx.x - row_blocks) * 4 + tid / 64;
    if (block >= p.b * blocks) return;
    const uint32_t batch = block / blocks, row = (block - batch * blocks) * 64 + (tid & 63);
    const Span mine = span_of(p, batch, min(row, p.nq - 1));
    Spans s;
    s.none();
    s.add(mine);
    s.over_lanes<63>();
    char* record = p.spans + (size_t)block * kSpanRecord;
    *reinterpret_cast<Span*>(record + 8 * (tid & 63)) = mine;
    if ((tid & 63) == 0) *reinterpret_cast<Spans*>(record + 64 * 8) = s;
  }
}

// Query tiles of TILE rows (TILE divides 64) that a tile of keys has to look at.
template <int TILE>
struct QueryTiles {
  const AttendParams& p;
  uint32_t batch;
  __device__ __forceinline__ const char* record(uint32_t tile) const {
    return p.spans + ((size_t)batch * ((p.nq + 63) / 64) + tile * TILE / 64) * kSpanRecord;
  }
  // without first and last
  __device__ __forceinline__ Spans computed(uint32_t tile) const {
    if (!p.causal) return Spans{0, 0, (int)p.nk, (int)p.nk};
    const int row0 = (int)(tile * TILE), row1 = min(row0 + TILE, (int)p.nq) - 1;
    const int least = min(max(row0 + p.shift + 1, 0), (int)p.nk), most = min(max(row1 + p.shift + 1, 0), (int)p.nk);
    return Spans{0, 0, least, most};
  }
  // tiles begin .. end - 1 hold every query that sees any of the keys k0 .. k1 - 1 (all threads of the workgroup call this)
  template <int THREADS>
  __device__ __forceinline__ void range(int k0, int k1, int* shared, uint32_t& begin, uint32_t& end) const {
    const uint32_t tiles = (p.nq + TILE - 1) / TILE;
    begin = 0;
    end = tiles;
    if (!p.spans) {
      if (p.causal) begin = min((uint32_t)max(k0 - p.shift, 0) / TILE, tiles);
      return;
    }
    if (threadIdx.x == 0) {
      shared[0] = (int)tiles;
      shared[1] = 0;
    }
    __syncthreads();
    int least = (int)tiles, most = 0;
    for (uint32_t t = threadIdx.x; t < tiles; t += THREADS) {
      const Spans s = *reinterpret_cast<const Spans*>(record(t) + 64 * 8);
      if (s.touches(k0, k1)) {
        least = min(least, (int)t);
        most = (int)t + 1;
      }
    }
    if (most > 0) {
      atomicMin(&shared[0], least);
      atomicMax(&shared[1], most);
    }
    __syncthreads();
    begin = (uint32_t)__builtin_amdgcn_readfirstlane(shared[0]);
    end = max(begin, (uint32_t)__builtin_amdgcn_readfirstlane(shared[1]));
  }
};

// A tile of 16 KB NW keys against the queries of all heads that share them.  GRAD: dk and dv (Q and dO tiles of BQ rows), else
// the keys' weights (Q tiles).  S = Q K^T with keys as columns: a lane has one key and four consecutive queries, P and dS are the
// right operands of dV^T += dO^T P and dK^T += Q^T dS as they are.  All that a tile of queries needs comes by transfers requested
// a tile ahead; a load into registers inside the loop would have to wait for them.
template <typename T, int DPAD, int DUSE, int BQ, int NW, int KB, bool GRAD>
__device__ __forceinline__ void keys_body(const AttendParams& p) {
  using L = Tile<T, DPAD, BQ>;
  constexpr int BK = 16 * KB * NW, KS = DUSE / 32, DT = DUSE / 16, TILES = GRAD ? 2 : 1;
  static_assert(64 % BQ == 0 && BQ % 32 == 0 && NW >= 3, "query tile");
  __shared__ __attribute__((aligned(1024))) char smem[2][TILES][L::BYTES];  // [buffer][Q, dO]
  __shared__ __attribute__((aligned(16))) float row_of[2][BQ][2];
  __shared__ __attribute__((aligned(16))) Span span_of_row[2][BQ];
  __shared__ __attribute__((aligned(16))) Spans spans_of_tile[2];
  __shared__ int shared_range[2];

  uint32_t head, at;
  xcd_map(blockIdx.x, p.tiles * p.parts, p.b * p.hkv, head, at);
  if (head >= p.b * p.hkv) return;
  const uint32_t tile = at / p.parts, part = at - tile * p.parts;
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int k0 = (int)(tile * BK), kw0 = k0 + wave * (16 * KB), kw1 = min(kw0 + 16 * KB, (int)p.nk);

  const T* K = (const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh;
  const T* V = (const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh;
  Frag<T> kf[KB][KS], vf[GRAD ? KB : 1][GRAD ? KS : 1];
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int64_t key = min(kw0 + 16 * b + r, (int)p.nk - 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t col = 32 * ks + 8 * g;
      kf[b][ks] = col < p.d ? load_frag<T>(K + key * p.k.sn + col) : zero_frag<T>();
      if constexpr (GRAD) vf[b][ks] = col < p.d ? load_frag<T>(V + key * p.v.sn + col) : zero_frag<T>();
    }
  }
  f32x4 dk[GRAD ? KB : 1][GRAD ? DT : 1], dv[GRAD ? KB : 1][GRAD ? DT : 1];
  float weight[KB];
#pragma unroll
  for (int b = 0; b < KB; ++b) weight[b] = 0.0f;
  if constexpr (GRAD) {
    clear_sums<T>(dk);
    clear_sums<T>(dv);
  }
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<2 * TILES * L::BYTES, 64 * NW>(&smem[0][0][0], tid);

  const QueryTiles<BQ> queries{p, batch};
  uint32_t begin, end;
  queries.template range<64 * NW>(k0, min(k0 + BK, (int)p.nk), shared_range, begin, end);
  // the walk: query tiles of the first head, of the second, ...; a part is a run of it
  const uint32_t per = end - begin, total = per * p.group;
  uint32_t item = (uint32_t)((uint64_t)total * part / p.parts);
  const uint32_t stop = (uint32_t)((uint64_t)total * (part + 1) / p.parts);

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[0][0][0]);
  const uint32_t lds_rows = lds_address(&row_of[0][0][0]), lds_spans = lds_address(&span_of_row[0][0]), lds_tile = lds_address(&spans_of_tile[0]);
  const typename L::template Requests<NW> of_q((uint32_t)(p.q.sn * sizeof(T)), p.d, wave, lane), of_g((uint32_t)(p.grad_o.sn * sizeof(T)), p.d, wave, lane);
  const uint32_t blocks = (p.nq + 63) / 64;
  auto place = [&](uint32_t n, uint32_t& hq, uint32_t& t) {
    const uint32_t h = n / per;
    hq = hkv * p.group + h;
    t = begin + (n - h * per);
  };
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

#pragma unroll
  for (int b = 0; b < KB; ++b) {
    arrive(kf[b]);
    if constexpr (GRAD) {
      arrive(vf[b]);
      keep(kf[b]);
      keep(vf[b]);
    }
  }
  int buf = 0;
  uint32_t hq = 0, t = 0, slope_of = 0xffffffff;
  float slope2 = 0.0f;
  if (item < stop) {
    __syncthreads();  // (the tile memory is clear)
    place(item, hq, t);
    request(hq, t, 0);
  }
  for (; item < stop; ++item, buf ^= 1) {
    const uint32_t this_t = t;
    if (p.slopes && hq != slope_of) {
      slope_of = hq;
      slope2 = p.slopes[hq] * Bend::I_LOG2_E;
      asm volatile("" : "+v"(slope2));
    }
    dma_wait_all();
    __syncthreads();
    if (item + 1 < stop) {
      place(item + 1, hq, t);
      request(hq, t, buf ^ 1);
    }
    Spans spans = queries.computed(this_t);
    if (p.spans) {
      spans = spans_of_tile[buf];
      spans.uniform();
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
      Frag<T> pf[KB], df[KB];
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
        if constexpr (GRAD) {
          settle_kept(s);
          settle_kept(dp);
        } else {
          settle(s);
        }
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
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            Span span{0, p.causal ? (int)(this_t * BQ) + row + i + p.shift + 1 : (int)p.nk};
            if (p.spans) span = span_of_row[buf][row + i];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              const int key = kw0 + 16 * b + r;
              if (key < span.first || key >= span.last) {
                s[b][i] = -INFINITY;
                dp[b][i] = 0.0f;
              }
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
              df[b][4 * h + i] = (T)(e * dp[b][i]);
            } else {
              weight[b] = __builtin_fmaf(e, other[i], weight[b]);
            }
          }
      }
      if constexpr (GRAD) {
        ready(pf);
        ready(df);
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
              add_mma(dk[b][step * COLS + c], col_q[step & 1][c], df[b]);
            }
        }
      }
    }
  }
  if constexpr (GRAD) {
    settled<T>(dk);
    settled<T>(dv);
  }

#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int key = kw0 + 16 * b + r;
    if constexpr (!GRAD) {
      const float sum = groups_sum(weight[b]);
      if (key >= (int)p.nk || g != 0) continue;
      const size_t to = (size_t)head * p.nk + key;
      if (p.parts > 1) p.partial_k[(size_t)part * p.b * p.hkv * p.nk + to] = sum;
      else p.weights_out[to] = p.weights_in ? p.weights_in[to] + sum : sum;
    } else {
      if (key >= (int)p.nk) continue;
      if (p.parts > 1) {
        const size_t to = (((size_t)part * p.b * p.hkv + head) * p.nk + key) * p.d;
#pragma unroll
        for (int c = 0; c < DT; ++c)
          if (16 * c + 4 * g < p.d) {
            store4(p.partial_k + to + 16 * c + 4 * g, dk[b][c] * p.scale);
            store4(p.partial_v + to + 16 * c + 4 * g, dv[b][c]);
          }
      } else {
        T* gk = (T*)p.grad_k.data + batch * p.grad_k.sb + hkv * p.grad_k.sh + key * p.grad_k.sn;
        T* gv = (T*)p.grad_v.data + batch * p.grad_v.sb + hkv * p.grad_v.sh + key * p.grad_v.sn;
#pragma unroll
        for (int c = 0; c < DT; ++c)
          if (16 * c + 4 * g < p.d) {
            store4(gk + 16 * c + 4 * g, dk[b][c] * p.scale);
            store4(gv + 16 * c + 4 * g, dv[b][c]);
          }
      }
    }
  }
}

// The parts of dk and dv added up in their order, four elements a work-item.
template <typename T>
__device__ __forceinline__ void join_gradients_body(const AttendParams& p) {
  const uint64_t part = (uint64_t)p.b * p.hkv * p.nk * p.d;
  const uint64_t fours = part / 4;
  for (uint64_t n = (uint64_t)blockIdx.x * 256 + threadIdx.x; n < 2 * fours; n += (uint64_t)gridDim.x * 256) {
    const bool of_v = n >= fours;
    const uint64_t at = 4 * (of_v ? n - fours : n);
    const float* from = (of_v ? p.partial_v : p.partial_k) + at;
    f32x4 sum = *reinterpret_cast<const f32x4*>(from);
    for (uint32_t s = 1; s < p.parts; ++s) sum += *reinterpret_cast<const f32x4*>(from + s * part);
    const uint64_t row = at / p.d;
    const uint32_t col = (uint32_t)(at - row * p.d), bh = (uint32_t)(row / p.nk), key = (uint32_t)(row - (uint64_t)bh * p.nk);
    const uint32_t batch = bh / p.hkv, hkv = bh - batch * p.hkv;
    const AttendOperand& to = of_v ? p.grad_v : p.grad_k;
    store4((T*)to.data + batch * to.sb + hkv * to.sh + key * to.sn + col, sum);
  }
}

__device__ __forceinline__ void join_weights_body(const AttendParams& p) {
  const uint64_t count = (uint64_t)p.b * p.hkv * p.nk;
  for (uint64_t n = (uint64_t)blockIdx.x * 256 + threadIdx.x; n < count; n += (uint64_t)gridDim.x * 256) {
    float sum = 0.0f;
    for (uint32_t s = 0; s < p.parts; ++s) sum += p.partial_k[s * count + n];
    p.weights_out[n] = p.weights_in ? p.weights_in[n] + sum : sum;
  }
}

// dq of 16 QB NW queries: the forward kernel's walk with two products of a tile (scores, dO V^T) and dQ^T += K^T dS^T.
template <typename T, int DPAD, int DUSE, int BN, int NW, int QB>
__device__ __forceinline__ void queries_body(const AttendParams& p) {
  using L = Tile<T, DPAD, BN>;
  constexpr int BM = 16 * QB * NW, KS = DUSE / 32, DT = DUSE / 16;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ Spans shared_spans[NW];

  uint32_t head, tile;
  xcd_map(blockIdx.x, p.tiles, p.b * p.hq, head, tile);
  if (head >= p.b * p.hq) return;
  if (p.causal) tile = p.tiles - 1 - tile;
  const uint32_t batch = head / p.hq, hq = head - batch * p.hq, hkv = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t row0 = tile * BM + wave * (16 * QB);

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
  }
  mine.over_lanes<15>();
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
      if (!mine.touches(k0, k0 + BN)) continue;
      const bool whole = mine.whole(k0, k0 + BN);
      const char* tk = &smem[buf][0][0];
      const char* tv = &smem[buf][1][0];
#pragma unroll
      for (int u = 0; u < BN / 32; ++u) {
        Frag<T> df[QB];
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
          settle(s);
          settle(dp);
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
              const float away = (float)((int)(row0 + 16 * b) + r + p.shift - k0 - 16 * block - 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i) s[b][i] = __builtin_fmaf(-slope2, fabsf(away - (float)i), s[b][i]);
            }
          }
          if (!whole) {
#pragma unroll
            for (int b = 0; b < QB; ++b) {
              const uint32_t seen = (uint32_t)max(span[b].last - span[b].first, 0);
              const int at = k0 + 16 * block + 4 * g - span[b].first;
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
            for (int i = 0; i < 4; ++i) df[b][4 * h + i] = (T)(fast_exp2(__builtin_fmaf(s[b][i], bend.mult, -lse[b])) * dp[b][i]);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const Frag<T> a = reader.across(tk, t, u);
#pragma unroll
          for (int b = 0; b < QB; ++b) dq[b][t] = mma(a, df[b], dq[b][t]);
        }
      }
    }
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

}  // namespace attend
