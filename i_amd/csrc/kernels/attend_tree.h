// Attention of a few query rows (the nodes of a tree of drafted tokens, or one token) against a long cache in pages.
//
// The time is that of reading the cache.  A workgroup takes a part of one key head's keys and 16 RT of its query rows (the rows
// are the nodes of all query heads that share the key head).  Its wavefronts walk tiles of 32 keys of their own, each with two
// tiles of K and V in LDS and no barrier between them: while one tile is worked on the next is on its way, 64 KiB and more a
// compute unit.  Where the rows of the tiles lie in memory is looked up once at the start, for the whole part.  The
// wavefronts' results are put together in LDS, those of the parts by a second launch, in the order of the keys.
#pragma once
#include "attend.h"

namespace attend {

constexpr int kTreePart = 1024;  // most keys of a part

// 16 bytes a lane from a 64-bit address of the lane's own (see dma16)
__device__ __forceinline__ void dma16_at(const void* at, uint32_t lds_base) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(at), "s"(__builtin_amdgcn_readfirstlane((int)lds_base))
      : "memory");
}

__device__ __forceinline__ uint32_t page_of(const AttendCache& c, uint32_t batch, uint32_t index) {
  if (!c.table) return batch < c.pages ? batch : 0;
  const uint32_t page = (uint32_t)c.table[(int64_t)batch * c.table_stride + index];
  return page < c.pages ? page : 0;
}

// slots of a sequence before its drafted tokens, and with them (of one sequence for all lanes)
__device__ __forceinline__ void tree_lengths(const TreeParams& p, uint32_t batch, uint32_t& length, uint32_t& total) {
  const int given = p.lengths[batch];
  const uint32_t most = p.max_length - p.nodes;
  length = given < 0 ? 0 : min((uint32_t)given, most);
  length = (uint32_t)__builtin_amdgcn_readfirstlane((int)length);
  total = length + p.nodes;
}

template <typename T, int DPAD, int DUSE, int NW, int RT>
__device__ __forceinline__ void tree_body(const TreeParams& p) {
  using L = Tile<T, DPAD, 32>;
  constexpr int DT = DUSE / 16, THREADS = 64 * NW, LOADS = 2 * L::WL;
  static_assert(16 * RT * DPAD * 4 <= 4 * L::BYTES, "a wavefront's result fits its tiles");
  __shared__ __attribute__((aligned(1024))) char smem[NW][2][2][L::BYTES];  // [wavefront][buffer][K, V]
  __shared__ int64_t offset_of[kTreePart][2];  // where a key's rows of K and V lie, in bytes
  __shared__ __attribute__((aligned(16))) int position_of[kTreePart];
  __shared__ float shared_m[NW][16 * RT], shared_l[NW][16 * RT];

  // parts of one key head beside each other on an XCD, the row tiles of a part next to each other
  uint32_t head, at;
  xcd_map(blockIdx.x, p.parts * p.row_tiles, p.b * p.hkv, head, at);
  if (head >= p.b * p.hkv) return;
  const uint32_t part = at / p.row_tiles, row_tile = at - part * p.row_tiles;
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv;
  uint32_t length, total;
  tree_lengths(p, batch, length, total);
  const uint32_t c0 = part * p.chunk, c1 = min(c0 + p.chunk, total);
  if (c0 >= c1) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int start = p.start ? p.start[batch] : (int)length;
  const uint64_t* visible = p.visible ? p.visible + (int64_t)batch * p.visible_stride : nullptr;

  for (uint32_t i = tid; i < c1 - c0; i += THREADS) {
    const uint32_t key = c0 + i, index = key / p.cache.page, slot = key - index * p.cache.page;
    const int64_t page = page_of(p.cache, batch, index);
    offset_of[i][0] = (page * p.cache.k_page + hkv * p.cache.k_head + slot * p.cache.k_slot) * (int64_t)sizeof(T);
    offset_of[i][1] = (page * p.cache.v_page + hkv * p.cache.v_head + slot * p.cache.v_slot) * (int64_t)sizeof(T);
    if (p.slopes) {
      int position = p.positions && key < length ? p.positions[(int64_t)head * p.positions_stride + key] : (int)key;
      if (key >= length) {
        const uint64_t word = visible ? visible[key - length] : (2ull << (key - length)) - 1;
        position = start + __popcll(word) - 1;
      }
      position_of[i] = position;
    }
  }
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<NW * 4 * L::BYTES, THREADS>(&smem[0][0][0][0], tid);

  Rows<T, DPAD, DUSE, RT> rows;
  rows.clear();
  uint64_t word[RT];
  float slope2[RT];
  int position[RT];
  int64_t score_at[RT];  // where the scores of a counted row go, -1: not kept
#pragma unroll
  for (int b = 0; b < RT; ++b) {
    const uint32_t row = row_tile * (16 * RT) + 16 * b + r, inside = min(row, p.rows - 1);
    const uint32_t hg = inside / p.nodes, node = inside - hg * p.nodes, hq = hkv * p.group + hg;
    rows.load_q(b, (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh + node * p.q.sn, true, p.d, g);
    word[b] = visible ? visible[node] : (2ull << node) - 1;
    slope2[b] = p.slopes ? p.slopes[hq] * Bend::I_LOG2_E : 0.0f;
    position[b] = start + __popcll(word[b]) - 1;
    score_at[b] = -1;
    if (p.scores && row < p.rows && (p.counted >> node & 1))
      score_at[b] = ((int64_t)head * p.group * p.counted_nodes + hg * p.counted_nodes + __popcll(p.counted & ((1ull << node) - 1))) * ((int64_t)p.parts * p.chunk);
  }
#pragma unroll
  for (int b = 0; b < RT; ++b) arrive(rows.q[b]);
  __syncthreads();

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[wave][0][0][0]), chunks = p.d * sizeof(T) / 16;
  auto request = [&](uint32_t k0, int buf) {
#pragma unroll
    for (int w = 0; w < L::WL; ++w) {
      const uint32_t row = w * L::RPW + lane / L::CH;
      const uint32_t chunk = (lane % L::CH) ^ L::swizzle(row);
      const uint32_t key = min(k0 + row, c1 - 1) - c0;
      // (a wave-load holds whole rows, so some lane always takes part and the count of transfers in flight is known)
      if (chunk < chunks) {
        dma16_at((const char*)p.cache.k + offset_of[key][0] + 16 * chunk, lds + (2 * buf) * L::BYTES + 1024 * w);
        dma16_at((const char*)p.cache.v + offset_of[key][1] + 16 * chunk, lds + (2 * buf + 1) * L::BYTES + 1024 * w);
      }
    }
  };
  uint32_t k0 = c0 + 32 * wave;
  if (k0 < c1) {
    request(k0, 0);
    for (int buf = 0; k0 < c1; k0 += 32 * NW, buf ^= 1) {
      if (k0 + 32 * NW < c1) {
        // every read of the tile before is answered; the transfers of this tile are done when only the next one's are under way
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request(k0 + 32 * NW, buf ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS < 63 ? LOADS : 63) : "memory");
      } else {
        dma_wait_all();
      }
      const bool whole = k0 + 32 <= min(length, c1);
      rows.template tile<2>(&smem[wave][buf][0][0], &smem[wave][buf][1][0], bend, whole && !p.slopes && !p.scores, [&](f32x4 (&x)[RT][2]) {
        if (p.slopes) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const i32x4 of = *reinterpret_cast<const i32x4*>(&position_of[k0 - c0 + 16 * t + 4 * g]);
#pragma unroll
            for (int b = 0; b < RT; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) x[b][t][i] = __builtin_fmaf(-slope2[b], fabsf((float)(position[b] - of[i])), x[b][t][i]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t key = k0 + 16 * t + 4 * g + i;
              const uint32_t node = key - length;  // (key < length: the prefix, seen by all)
#pragma unroll
              for (int b = 0; b < RT; ++b)
                if (key >= c1 || (key >= length && !(word[b] >> (node & 63) & 1))) x[b][t][i] = -INFINITY;
            }
        }
        if (p.scores) {
#pragma unroll
          for (int b = 0; b < RT; ++b)
            if (score_at[b] >= 0) {
#pragma unroll
              for (int t = 0; t < 2; ++t) store4(p.scores + score_at[b] + k0 + 16 * t + 4 * g, x[b][t]);
            }
        }
      }, reader);
    }
  }

  // the wavefronts' results: 16-byte chunk c of row w at chunk c ^ (w & 15)
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(&smem[wave][0][0][0]);
#pragma unroll
  for (int b = 0; b < RT; ++b) {
    const float sum = groups_sum(rows.l[b]);
    if (g == 0) {
      shared_m[wave][16 * b + r] = rows.m[b];
      shared_l[wave][16 * b + r] = sum;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) store4(mine + (16 * b + r) * DPAD + 4 * ((4 * t + g) ^ r), rows.o[b][t]);
  }
  __syncthreads();
  const uint32_t fours = p.d / 4;
  for (uint32_t i = tid; i < 16 * RT * fours; i += THREADS) {
    const uint32_t row = i / fours, c = i - row * fours, to = row_tile * (16 * RT) + row;
    if (to >= p.rows) break;
    float top = shared_m[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, shared_m[w][row]);
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = shared_m[w][row], weigh = m == -INFINITY ? 0.0f : fast_exp2(m - top);
      sum += weigh * shared_l[w][row];
      // (a wavefront that had no tile leaves zeros)
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(&smem[w][0][0][0]) + row * DPAD + 4 * (c ^ (row & 15))) * weigh;
    }
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const float lse = top == -INFINITY ? -INFINITY : top + __builtin_amdgcn_logf(sum);
    const size_t partial = ((size_t)head * p.parts + part) * p.rows + to;
    if (c == 0 && p.partial_lse) p.partial_lse[partial] = lse;
    if (p.parts > 1) {
      store4(p.partial_o + partial * p.d + 4 * c, o);
    } else {
      const uint32_t hg = to / p.nodes, node = to - hg * p.nodes, hq = hkv * p.group + hg;
      store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + 4 * c, o);
      if (c == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = lse * 0.69314718056f;
    }
  }
}

// The parts of a row put together (a wavefront per row), then the weights of the keys: exp(score - lse) over the counted rows.
template <typename T>
__device__ __forceinline__ void tree_join_body(const TreeParams& p) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t join_blocks = p.parts > 1 ? (p.b * p.hkv * p.rows + 3) / 4 : 0;
  uint32_t length, total;
  if (blockIdx.x < join_blocks) {
    const uint32_t at = blockIdx.x * 4 + tid / 64;
    if (at >= p.b * p.hkv * p.rows) return;
    const uint32_t head = at / p.rows, row = at - head * p.rows, batch = head / p.hkv, hkv = head - batch * p.hkv;
    tree_lengths(p, batch, length, total);
    const uint32_t live = (total + p.chunk - 1) / p.chunk;
    const float* lse = p.partial_lse + (size_t)head * p.parts * p.rows + row;
    const float* from = p.partial_o + ((size_t)head * p.parts * p.rows + row) * p.d;
    float top = -INFINITY;
    for (uint32_t s = lane; s < live; s += 64) top = fmaxf(top, lse[(size_t)s * p.rows]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
    for (uint32_t s0 = 0; s0 < live; s0 += 64) {
      const float mine = s0 + lane < live ? fast_exp2(lse[(size_t)(s0 + lane) * p.rows] - ref) : 0.0f;
      sum += mine;
      const uint32_t here = min(live - s0, 64u);
#pragma unroll 4
      for (uint32_t s = 0; s < here; ++s) {
        const float weigh = __shfl(mine, (int)s);
        if (4 * lane < p.d) o += *reinterpret_cast<const f32x4*>(from + (size_t)(s0 + s) * p.rows * p.d + 4 * lane) * weigh;
      }
    }
    sum = wave_sum(sum);
    const uint32_t hg = row / p.nodes, node = row - hg * p.nodes, hq = hkv * p.group + hg;
    if (4 * lane < p.d) store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + 4 * lane, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (lane == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = top == -INFINITY ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
    return;
  }
  // 256 keys of one key head
  __shared__ float shared_lse[256];
  const uint32_t tiles = (p.max_length + 255) / 256, at = blockIdx.x - join_blocks;
  const uint32_t head = at / tiles, key = (at - head * tiles) * 256 + tid, batch = head / p.hkv;
  if (head >= p.b * p.hkv) return;
  tree_lengths(p, batch, length, total);
  const uint32_t live = (total + p.chunk - 1) / p.chunk, counted = p.group * p.counted_nodes;
  const int64_t stride = (int64_t)p.parts * p.chunk;
  const float* scores = p.scores + (int64_t)head * counted * stride + key;
  float sum = 0.0f;
  for (uint32_t first = 0; first < counted; first += 256) {
    __syncthreads();
    if (first + tid < counted) {
      // counted row n: head n / counted_nodes of the group, the (n % counted_nodes)-th of the counted nodes
      const uint32_t n = first + tid, hg = n / p.counted_nodes;
      uint64_t left = p.counted;
      for (uint32_t k = n - hg * p.counted_nodes; k > 0; --k) left &= left - 1;
      const uint32_t row = hg * p.nodes + __builtin_ctzll(left);
      const float* lse = p.partial_lse + (size_t)head * p.parts * p.rows + row;
      float top = -INFINITY, all = 0.0f;
      for (uint32_t s = 0; s < live; ++s) top = fmaxf(top, lse[(size_t)s * p.rows]);
      const float ref = top == -INFINITY ? 0.0f : top;
      for (uint32_t s = 0; s < live; ++s) all += fast_exp2(lse[(size_t)s * p.rows] - ref);
      shared_lse[tid] = top == -INFINITY ? INFINITY : top + __builtin_amdgcn_logf(all);
    }
    __syncthreads();
    if (key < total) {
      const uint32_t here = min(counted - first, 256u);
#pragma unroll 4
      for (uint32_t n = 0; n < here; ++n) sum += fast_exp2(scores[(int64_t)(first + n) * stride] - shared_lse[n]);
    }
  }
  if (key < p.max_length) {
    const float before = p.weights_in[(int64_t)head * p.weights_in_stride + key];
    p.weights_out[(int64_t)head * p.weights_out_stride + key] = before + sum;
  }
}

}  // namespace attend
