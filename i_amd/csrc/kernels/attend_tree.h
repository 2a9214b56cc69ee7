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

constexpr int kTreePart = 1024, kTreeRowsPart = 512;  // most keys of a part

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

// Where the rows of keys c0 .. c1 - 1 lie, in bytes from the cache's start, and (for a bias) their positions; by THREADS threads.
template <typename T, int THREADS>
__device__ __forceinline__ void look_up(const TreeParams& p, uint32_t batch, uint32_t hkv, uint32_t head, uint32_t length, int start, uint32_t c0, uint32_t c1,
                                        int64_t (*offset_of)[2], int* position_of) {
  const uint64_t* visible = p.visible ? p.visible + (int64_t)batch * p.visible_stride : nullptr;
  for (uint32_t i = threadIdx.x; i < c1 - c0; i += THREADS) {
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
}

// A query row: node `row % nodes` of the (row / nodes)-th query head of a key head.  (A row past the end repeats the last one.)
struct TreeRow {
  uint32_t hq, node;
  uint64_t word;     // the nodes that it sees
  float slope2;
  int position;
  int64_t score_at;  // where the scores of a counted row go, -1: not kept
  __device__ __forceinline__ void set(const TreeParams& p, uint32_t batch, uint32_t head, uint32_t hkv, uint32_t row, int start) {
    const uint32_t inside = min(row, p.rows - 1), hg = inside / p.nodes;
    node = inside - hg * p.nodes;
    hq = hkv * p.group + hg;
    word = p.visible ? p.visible[(int64_t)batch * p.visible_stride + node] : (2ull << node) - 1;
    slope2 = p.slopes ? p.slopes[hq] * Bend::I_LOG2_E : 0.0f;
    position = start + __popcll(word) - 1;
    score_at = -1;
    if (p.scores && row < p.rows && (p.counted >> node & 1))
      score_at = ((int64_t)head * p.group * p.counted_nodes + hg * p.counted_nodes + __popcll(p.counted & ((1ull << node) - 1))) * ((int64_t)p.parts * p.chunk);
  }
  template <typename T>
  __device__ __forceinline__ const T* q(const TreeParams& p, uint32_t batch) const {
    return (const T*)p.q.data + batch * p.q.sb + hq * p.q.sh + node * p.q.sn;
  }
};

// Bias, mask and, where they are wanted, a copy of the scores of keys k0 .. k0 + 16 KT - 1.
template <int QB, int KT>
__device__ __forceinline__ void finish_scores(const TreeParams& p, f32x4 (&x)[QB][KT], const TreeRow* of, const int* position_of, uint32_t k0, uint32_t c0,
                                              uint32_t c1, uint32_t length, bool whole, int g) {
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    if (p.slopes) {
      const i32x4 at = *reinterpret_cast<const i32x4*>(&position_of[k0 - c0 + 16 * t + 4 * g]);
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[b][t][i] = __builtin_fmaf(-of[b].slope2, fabsf((float)(of[b].position - at[i])), x[b][t][i]);
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t key = k0 + 16 * t + 4 * g + i;
        const uint32_t node = key - length;  // (key < length: the prefix, seen by all)
#pragma unroll
        for (int b = 0; b < QB; ++b)
          if (key >= c1 || (key >= length && !(of[b].word >> (node & 63) & 1))) x[b][t][i] = -INFINITY;
      }
    }
    if (p.scores) {
#pragma unroll
      for (int b = 0; b < QB; ++b)
        if (of[b].score_at >= 0) store4(p.scores + of[b].score_at + k0 + 16 * t + 4 * g, x[b][t]);
    }
  }
}

// four outputs of a row and the logarithm of its sum (base 2): to the partial results, or where a part is all there is to the end
template <typename T>
__device__ __forceinline__ void give_row(const TreeParams& p, uint32_t head, uint32_t part, uint32_t row, uint32_t column, f32x4 o, float lse) {
  const size_t partial = ((size_t)head * p.parts + part) * p.rows + row;
  if (column == 0 && p.partial_lse) p.partial_lse[partial] = lse;
  if (p.parts > 1) {
    store4(p.partial_o + partial * p.d + column, o);
    return;
  }
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv, hg = row / p.nodes, node = row - hg * p.nodes, hq = hkv * p.group + hg;
  store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + column, o);
  if (column == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = lse * 0.69314718056f;
}

template <typename T, int DPAD, int DUSE, int NW, int RT>
__device__ __forceinline__ void tree_body(const TreeParams& p) {
  using L = Tile<T, DPAD, 32>;
  constexpr int THREADS = 64 * NW, LOADS = 2 * L::WL;
  static_assert(16 * RT * DPAD * 4 <= 4 * L::BYTES, "a wavefront's result fits its tiles");
  __shared__ __attribute__((aligned(1024))) char smem[NW][2][2][L::BYTES];  // [wavefront][buffer][K, V]
  __shared__ int64_t offset_of[kTreePart][2];
  __shared__ __attribute__((aligned(16))) int position_of[kTreePart];
  __shared__ Merge<NW, RT> shared;

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
  look_up<T, THREADS>(p, batch, hkv, head, length, start, c0, c1, offset_of, position_of);
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<NW * 4 * L::BYTES, THREADS>(&smem[0][0][0][0], tid);

  Rows<T, DPAD, DUSE, RT> rows;
  rows.clear();
  TreeRow of[RT];
#pragma unroll
  for (int b = 0; b < RT; ++b) {
    of[b].set(p, batch, head, hkv, row_tile * (16 * RT) + 16 * b + r, start);
    rows.load_q(b, of[b].template q<T>(p, batch), true, p.d, g);
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
        finish_scores<RT, 2>(p, x, of, position_of, k0, c0, c1, length, whole, g);
      }, reader);
    }
  }

  merge_rows(rows, shared, &smem[0][0][0][0], 4 * L::BYTES, p.d, min(16u * RT, p.rows - row_tile * (16 * RT)), [&](uint32_t n, uint32_t column, f32x4 o, float lse) {
    give_row<T>(p, head, part, row_tile * (16 * RT) + n, column, o, lse);
  });
}

// The same for more rows: 64 a workgroup, 16 of each of its four wavefronts, all of them on the same tile of BN keys; a barrier a tile.
template <typename T, int DPAD, int DUSE, int BN>
__device__ __forceinline__ void tree_rows_body(const TreeParams& p) {
  using L = Tile<T, DPAD, BN>;
  constexpr int NW = 4, KT = BN / 16, EACH = (L::WL + NW - 1) / NW;
  static_assert(L::WL % NW == 0, "tile shape");
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ int64_t offset_of[kTreeRowsPart][2];
  __shared__ __attribute__((aligned(16))) int position_of[kTreeRowsPart];

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
  look_up<T, 64 * NW>(p, batch, hkv, head, length, start, c0, c1, offset_of, position_of);
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<4 * L::BYTES, 64 * NW>(&smem[0][0][0], tid);

  Rows<T, DPAD, DUSE, 1> rows;
  rows.clear();
  const uint32_t row = row_tile * 64 + 16 * wave + r;
  TreeRow mine;
  mine.set(p, batch, head, hkv, row, start);
  rows.load_q(0, mine.template q<T>(p, batch), true, p.d, g);
  arrive(rows.q[0]);
  __syncthreads();

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[0][0][0]), chunks = p.d * sizeof(T) / 16;
  auto request = [&](uint32_t k0, int buf) {
#pragma unroll
    for (int it = 0; it < EACH; ++it) {
      const uint32_t w = wave + NW * it, in_tile = w * L::RPW + lane / L::CH;
      const uint32_t chunk = (lane % L::CH) ^ L::swizzle(in_tile);
      const uint32_t key = min(k0 + in_tile, c1 - 1) - c0;
      if (chunk < chunks) {
        dma16_at((const char*)p.cache.k + offset_of[key][0] + 16 * chunk, lds + (2 * buf) * L::BYTES + 1024 * w);
        dma16_at((const char*)p.cache.v + offset_of[key][1] + 16 * chunk, lds + (2 * buf + 1) * L::BYTES + 1024 * w);
      }
    }
  };
  request(c0, 0);
  int buf = 0;
  for (uint32_t k0 = c0; k0 < c1; k0 += BN, buf ^= 1) {
    dma_wait_all();
    __syncthreads();
    if (k0 + BN < c1) request(k0 + BN, buf ^ 1);
    const bool whole = k0 + BN <= min(length, c1);
    rows.template tile<KT>(&smem[buf][0][0], &smem[buf][1][0], bend, whole && !p.slopes && !p.scores, [&](f32x4 (&x)[1][KT]) {
      finish_scores<1, KT>(p, x, &mine, position_of, k0, c0, c1, length, whole, g);
    }, reader);
  }
  const float sum = groups_sum(rows.l[0]);
  if (row >= p.rows) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, lse = rows.m[0] == -INFINITY ? -INFINITY : rows.m[0] + __builtin_amdgcn_logf(sum);
#pragma unroll
  for (int t = 0; t < DUSE / 16; ++t)
    if (16 * t + 4 * g < p.d) give_row<T>(p, head, part, row, 16 * t + 4 * g, rows.o[0][t] * inv, lse);
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
