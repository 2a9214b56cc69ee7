// Attention forward with masks, capped scores and a bias by distance.
//
// A workgroup of NW wavefronts takes 16 QB NW queries of one head, a wavefront 16 QB of them, one query per lane column:
// S^T = K Q^T, O^T += V^T P^T (attend.h).  K and V tiles of BN keys are transferred into one half of the tile memory while
// the other half is worked on; one barrier a tile.  The keys walked are those between the least `first` and the largest `last` of
// the workgroup's queries; a wavefront leaves out the tiles that none of its own queries sees and tests scores one by one only in
// tiles that some of its queries see in part.
//
// What keys that no query sees hold does not matter, NaN and infinities included: those outside the walked range are never read (their
// rows are replaced by the nearest one inside), those that first and last leave out in between are set to zero (unseen_keys).
// Without first and last there is nothing in between.
//
// Bound by the wavefronts' own chains: two wavefronts a SIMD read every operand of a tile from LDS (half of LDS's time), multiply
// (two fifths of the matrix units') and take exponentials, and none of the three is busy all the time.  32 rows a wavefront, since a tile's
// LDS reads serve all of them (with 16 it takes 1.28 times as long); 64 keys a step, since a step has a cost of its own (with 32 keys
// in four buffers 1.17 times).  Measured, 128 columns of bf16, call after call: 2 x 16 heads of 4096, all keys, 264 us, 1040 TFLOP/s; causal 181 us;
// f32, 1 x 16 heads of 2048 296 us, 116 TFLOP/s.  (The first calls after a pause take up to 1.3 times as long, at a lower clock.)
#pragma once
#include "attend.h"

namespace attend {

// HALVES 2: NW wavefronts for 16 QB NW / 2 queries, of which the second half of them takes the second half of every tile's keys; their
// results are put together at the end.  The walk of a workgroup is a chain of products, softmax, products and a barrier a tile that a
// lone wavefront on a SIMD spends mostly waiting; this halves it where there are not enough workgroups for two a SIMD (16 causal heads of
// 2048 x 128 bf16: 53 -> 44 us; 1024: 29.5 -> 19; f32 of 1024: 143 -> 79).
template <typename T, int DPAD, int DUSE, int BN, int NW, int QB, int HALVES = 1>
__device__ __forceinline__ void forward_body(const AttendParams& p) {
  using L = Tile<T, DPAD, BN>;
  constexpr int ROW_WAVES = NW / HALVES, BM = 16 * QB * ROW_WAVES, KEYS = BN / HALVES, KT = KEYS / 16, DT = DUSE / 16;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ Spans shared_spans[NW];
  __shared__ Span span_of_row[BM];

  uint32_t head, tile;
  xcd_map(blockIdx.x, p.tiles, p.b * p.hq, head, tile);
  if (head >= p.b * p.hq) return;
  // the queries that see most come first: a launch that ends on short ones ends evenly
  if (p.causal) tile = p.tiles - 1 - tile;
  const uint32_t batch = head / p.hq, hq = head - batch * p.hq, hkv = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int half = wave / ROW_WAVES, row_wave = wave % ROW_WAVES;
  const uint32_t row0 = tile * BM + row_wave * (16 * QB);

  const T* Q = (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh;
  const char* K = (const char*)((const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh);
  const char* V = (const char*)((const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh);

  Rows<T, DPAD, DUSE, QB> rows;
  Span span[QB];
  Spans mine;
  mine.none();
  rows.clear();
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const uint32_t row = min(row0 + 16 * b + r, p.nq - 1);  // (rows past the end repeat the last one and are not stored)
    rows.load_q(b, Q + row * p.q.sn, true, p.d, g);
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
  for (int b = 0; b < QB; ++b) arrive(rows.q[b]);
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
          clear_rows<L, NW>(&smem[buf][1][0], unseen, wave);
          __syncthreads();
        }
      }
      const int here = k0 + half * KEYS, in_tile = half * KEYS * L::RB;
      if (!mine.touches(here, here + KEYS)) continue;
      const bool whole = mine.whole(here, here + KEYS);
      rows.template tile<KT>(&smem[buf][0][in_tile], &smem[buf][1][in_tile], bend, whole && !p.slopes, [&](f32x4 (&x)[QB][KT]) {
        if (p.slopes) {
#pragma unroll
          for (int b = 0; b < QB; ++b) {
            const float away = (float)((int)(row0 + 16 * b) + r + p.shift - here - 4 * g);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int i = 0; i < 4; ++i) x[b][kt][i] = __builtin_fmaf(-slope2, fabsf(away - (float)(16 * kt + i)), x[b][kt][i]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int b = 0; b < QB; ++b) {
            const uint32_t seen = (uint32_t)max(span[b].last - span[b].first, 0);
            const int at = here + 4 * g - span[b].first;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if ((uint32_t)(at + 16 * kt + i) >= seen) x[b][kt][i] = -INFINITY;
          }
        }
      }, reader);
    }
  }

  if constexpr (HALVES == 2) {
    static_assert(ROW_WAVES * QB * DT * 1024 <= 4 * L::BYTES, "the results of a half fit the tiles");
    __shared__ float shared_m[ROW_WAVES][QB][16], shared_l[ROW_WAVES][QB][64];
    char* const left = &smem[0][0][0] + row_wave * (QB * DT * 1024) + 16 * lane;
    __syncthreads();
    if (half == 1) {
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        if (g == 0) shared_m[row_wave][b][r] = rows.m[b];
        shared_l[row_wave][b][lane] = rows.l[b];
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(left + 1024 * (b * DT + t)) = rows.o[b][t];
      }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const float other = shared_m[row_wave][b][r], top = fmaxf(rows.m[b], other);
      const float weigh = rows.m[b] == -INFINITY ? 0.0f : fast_exp2(rows.m[b] - top), weigh_other = other == -INFINITY ? 0.0f : fast_exp2(other - top);
      rows.m[b] = top;
      rows.l[b] = rows.l[b] * weigh + shared_l[row_wave][b][lane] * weigh_other;
#pragma unroll
      for (int t = 0; t < DT; ++t) rows.o[b][t] = rows.o[b][t] * weigh + *reinterpret_cast<const f32x4*>(left + 1024 * (b * DT + t)) * weigh_other;
    }
  }
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const uint32_t row = row0 + 16 * b + r;
    const float sum = groups_sum(rows.l[b]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (row >= p.nq) continue;
    if (g == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nq + row] = rows.m[b] == -INFINITY ? -INFINITY : (rows.m[b] + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
    T* out = (T*)p.o.data + batch * p.o.sb + hq * p.o.sh + row * p.o.sn;
#pragma unroll
    for (int t = 0; t < DT; ++t)
      if (16 * t + 4 * g < p.d) store4(out + 16 * t + 4 * g, rows.o[b][t] * inv);
  }
}

// 16 queries of one head a workgroup, its NW wavefronts walking tiles of 32 keys of their own (every NW-th one each, two tiles of K and
// V in LDS, no barrier between them) and putting their results together at the end: for calls of few queries, whose time is
// that of a walk over the keys.  (4 heads of 333 x 64 f32: 11 us a call, 18 with 128 queries a workgroup.)
template <typename T, int DPAD, int DUSE, int NW>
__device__ __forceinline__ void forward_few_body(const AttendParams& p) {
  using L = Tile<T, DPAD, 32>;
  constexpr int LOADS = 2 * L::WL;
  __shared__ __attribute__((aligned(1024))) char smem[NW][2][2][L::BYTES];  // [wavefront][buffer][K, V]
  __shared__ Merge<NW, 1> shared;

  uint32_t head, tile;
  xcd_map(blockIdx.x, p.tiles, p.b * p.hq, head, tile);
  if (head >= p.b * p.hq) return;
  const uint32_t batch = head / p.hq, hq = head - batch * p.hq, hkv = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t row0 = 16 * tile, row = min(row0 + r, p.nq - 1);
  const char* K = (const char*)((const T*)p.k.data + batch * p.k.sb + hkv * p.k.sh);
  const char* V = (const char*)((const T*)p.v.data + batch * p.v.sb + hkv * p.v.sh);

  Rows<T, DPAD, DUSE, 1> rows;
  rows.clear();
  rows.load_q(0, (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh + row * p.q.sn, true, p.d, g);
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
  arrive(rows.q[0]);
  __syncthreads();
  int k0 = lo < hi ? lo / 32 * 32 + 32 * wave : hi;
  if (k0 < hi) {
    request(k0, 0);
    for (int buf = 0; k0 < hi; k0 += 32 * NW, buf ^= 1) {
      if (k0 + 32 * NW < hi) {
        // every read of the tile before is answered; the transfers of this tile are done when only the next one's are under way
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request(k0 + 32 * NW, buf ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS < 63 ? LOADS : 63) : "memory");
      } else {
        dma_wait_all();
      }
      const bool whole = all.whole(k0, k0 + 32);
      if (gap.touches(k0, k0 + 32)) {
        const uint64_t unseen = seen_keys(Span{lo, hi}, k0) & ~(uint64_t)row_or((uint32_t)seen_keys(span, k0)) & 0xffffffffu;
        if (unseen) clear_rows<L, 1>(&smem[wave][buf][1][0], unseen, 0);
      }
      rows.template tile<2>(&smem[wave][buf][0][0], &smem[wave][buf][1][0], bend, whole && !p.slopes, [&](f32x4 (&x)[1][2]) {
        const int at = k0 + 4 * g;
        if (p.slopes) {
          const float away = (float)((int)row0 + r + p.shift - at);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[0][t][i] = __builtin_fmaf(-slope2, fabsf(away - (float)(16 * t + i)), x[0][t][i]);
        }
        if (!whole) {
          const uint32_t seen = (uint32_t)max(span.last - span.first, 0);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((uint32_t)(at + 16 * t + i - span.first) >= seen) x[0][t][i] = -INFINITY;
        }
      }, reader);
    }
  }
  merge_rows(rows, shared, &smem[0][0][0][0], 4 * L::BYTES, p.d, min(16u, p.nq - row0), [&](uint32_t n, uint32_t column, f32x4 o, float lse) {
    store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + (row0 + n) * p.o.sn + column, o);
    if (column == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nq + row0 + n] = lse * 0.69314718056f;
  });
}

}  // namespace attend
