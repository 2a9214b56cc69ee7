// Attention of a few query rows (the nodes of a tree of drafted tokens, or one token) against a long cache in pages.
//
// The time is that of reading the cache.  The keys of all heads are dealt out in equal runs to as many workgroups as the chip holds
// at once, whatever the sequences' lengths are.  A workgroup has all query rows of a key head (the nodes of all query heads that
// share it) or, where there are many, a tile of them.  Its wavefronts walk tiles of 32 keys of their own, each with two tiles of K
// and V in LDS and no barrier between them: while one tile is worked on the next is on its way, 64 KiB a compute unit.  Where the
// pages lie is looked up once, for the whole run.  The wavefronts' results are put together in LDS, those of the runs by a second
// launch, in the order of the keys.
//
// Measured: 32 sequences of up to 8192 keys (8 heads of 128 bf16 columns, 506 MB), one token with weights: 112 us, 4.5 TB/s, and
// 10 for the join; in parts of 1024 keys 135 and 22.  8 trees of 48 nodes over 4096 keys, 4 query heads a key head: 44 us and 12, bound by
// the tiles' operand reads from LDS, which 32 rows a wavefront share (16 rows: 63).
#pragma once
#include "attend.h"

namespace attend {

constexpr int kTreePages = 512, kTreePositions = 1024;  // what a workgroup looks up at once: pages, and positions of keys for a bias

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

// a page to read: one that the cache does not have is page 0; a page to write: -1 then
__device__ __forceinline__ int64_t page_if_any(const AttendCache& c, uint32_t batch, uint32_t index) {
  const uint32_t page = c.table ? (uint32_t)c.table[(int64_t)batch * c.table_stride + index] : batch;
  return page < c.pages ? (int64_t)page : -1;
}
__device__ __forceinline__ uint32_t page_of(const AttendCache& c, uint32_t batch, uint32_t index) {
  return (uint32_t)max(page_if_any(c, batch, index), (int64_t)0);
}

// slots of a sequence before its drafted tokens, and with them (of one sequence for all lanes)
__device__ __forceinline__ void tree_lengths(const TreeParams& p, uint32_t batch, uint32_t& length, uint32_t& total) {
  const int given = p.lengths[batch];
  const uint32_t most = p.max_length - p.nodes;
  length = given < 0 ? 0 : min((uint32_t)given, most);
  length = (uint32_t)__builtin_amdgcn_readfirstlane((int)length);
  total = length + p.nodes;
}

// The work: the units (p.unit keys) of all key heads in a row, a sequence's heads beside each other, dealt out in equal runs.  All of
// it is of a whole wavefront; a lane keeps the length of one of the first 64 sequences.
struct TreeWork {
  const TreeParams& p;
  int kept;
  uint32_t total;  // units
  __device__ __forceinline__ uint32_t length_of(int given) const { return given < 0 ? 0 : min((uint32_t)given, p.max_length - p.nodes); }
  __device__ __forceinline__ uint32_t units(uint32_t length) const { return (length + p.nodes + p.unit - 1) / p.unit; }
  __device__ __forceinline__ uint32_t units_at(uint32_t i) const { return i < p.b ? units(length_of(i < 64 ? kept : p.lengths[i])) : 0; }
  __device__ __forceinline__ explicit TreeWork(const TreeParams& p) : p(p) {
    const uint32_t lane = threadIdx.x & 63;
    kept = p.lengths[min(lane, p.b - 1)];
    uint32_t mine = 0;
    for (uint32_t i = lane; i < p.b; i += 64) mine += units_at(i);
#pragma unroll
    for (int bit = 1; bit < 64; bit <<= 1) mine += (uint32_t)__shfl_xor((int)mine, bit);
    total = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine) * p.hkv;
  }
  // the sequence of a unit, how many units lie before it, and its length
  __device__ __forceinline__ void find(uint32_t unit, uint32_t& batch, uint32_t& before, uint32_t& length) const {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0;
    for (uint32_t b0 = 0;; b0 += 64) {
      const uint32_t mine = units_at(b0 + lane) * p.hkv;
      uint32_t upto = mine;
#pragma unroll
      for (int bit = 1; bit < 64; bit <<= 1) {
        const int other = __shfl_up((int)upto, bit);
        if ((int)lane >= bit) upto += (uint32_t)other;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > unit);
      if (past || b0 + 64 >= p.b) {
        const int at = past ? __builtin_ctzll(past) : 0;
        batch = b0 + at;
        before = base + (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), at);
        length = length_of(b0 == 0 ? __builtin_amdgcn_readlane(kept, at) : __builtin_amdgcn_readfirstlane(p.lengths[batch]));
        return;
      }
      base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
  }
};

// the key head that a run is at, and its units' number
struct TreeHead {
  uint32_t batch, hkv, head, begin, end;  // units begin .. end of all
  uint32_t length, total;                 // keys
  __device__ __forceinline__ void set(const TreeParams& p, uint32_t b, uint32_t h, uint32_t at) {
    batch = b;
    hkv = h;
    head = b * p.hkv + h;
    begin = at;
    end = at + (total + p.unit - 1) / p.unit;
  }
  __device__ __forceinline__ void at_unit(const TreeParams& p, const TreeWork& work, uint32_t unit) {
    uint32_t b, before;
    work.find(unit, b, before, length);
    total = length + p.nodes;
    const uint32_t each = work.units(length), h = (unit - before) / each;
    set(p, b, h, before + h * each);
  }
  __device__ __forceinline__ void next(const TreeParams& p) {
    if (hkv + 1 < p.hkv) return set(p, batch, hkv + 1, end);
    tree_lengths(p, batch + 1, length, total);
    set(p, batch + 1, 0, end);
  }
};

// The units from .. to - 1 of a workgroup; false: there are none.
__device__ __forceinline__ bool tree_run(const TreeParams& p, uint32_t run, TreeHead& head, uint32_t& from, uint32_t& to) {
  if (p.whole_heads) {
    if (run >= p.runs) return false;
    const uint32_t batch = run / p.hkv;
    tree_lengths(p, batch, head.length, head.total);
    head.set(p, batch, run - batch * p.hkv, 0);
    from = 0;
    to = head.end;
    return true;
  }
  const TreeWork work(p);
  const Deal deal(work.total, p.runs);
  if (run >= deal.shares) return false;
  from = deal.begin(run);
  to = deal.begin(run + 1);
  head.at_unit(p, work, from);
  return true;
}

// Nodes whose slots no node of the tree sees, and past which all of them are: a key past a sequence's end repeats its last slot.
__device__ __forceinline__ uint64_t unseen_nodes(const TreeParams& p, uint32_t batch) {
  if (!p.visible) return 0;
  const uint64_t unseen = ~wave_or(p.visible[(int64_t)batch * p.visible_stride + min((uint32_t)lane_now(), p.nodes - 1)]);
  const uint64_t nodes = p.nodes < 64 ? (1ull << p.nodes) - 1 : ~0ull;
  return unseen & nodes ? unseen | ~nodes : 0;
}

// Where the pages of keys c0 .. lie, and (for a bias) the positions of the keys.
struct TreeLookup {
  uint64_t page_at[kTreePages][2];  // address of a page's rows of the key head
  __attribute__((aligned(16))) int position_of[kTreePositions];
  uint64_t unseen;  // see unseen_nodes

  // looks up as much as there is room for, by THREADS threads between two barriers; returns the end of it (whole units, or c1)
  template <typename T, int THREADS>
  __device__ __forceinline__ uint32_t fill(const TreeParams& p, const TreeHead& h, int start, uint32_t c0, uint32_t c1) {
    const uint32_t first = page_index(p, c0);
    uint64_t most = (uint64_t)(first + kTreePages) * p.cache.page - c0;
    if (p.slopes) most = min(most, (uint64_t)kTreePositions);
    if (most < c1 - c0) c1 = c0 + (uint32_t)most / p.unit * p.unit;
    const uint32_t pages = page_index(p, c1 - 1) - first + 1;
    __syncthreads();
    if (threadIdx.x < 64) {
      const uint64_t nodes = unseen_nodes(p, h.batch);
      if (threadIdx.x == 0) unseen = nodes;
    }
    for (uint32_t i = threadIdx.x; i < pages; i += THREADS) {
      const int64_t page = page_of(p.cache, h.batch, first + i);
      page_at[i][0] = (uint64_t)p.cache.k + (uint64_t)(page * p.cache.k_page + h.hkv * p.cache.k_head) * sizeof(T);
      page_at[i][1] = (uint64_t)p.cache.v + (uint64_t)(page * p.cache.v_page + h.hkv * p.cache.v_head) * sizeof(T);
    }
    if (p.slopes) {
      const uint64_t* visible = p.visible ? p.visible + (int64_t)h.batch * p.visible_stride : nullptr;
      for (uint32_t i = threadIdx.x; i < c1 - c0; i += THREADS) {
        const uint32_t key = c0 + i;
        int position = p.positions && key < h.length ? p.positions[(int64_t)h.head * p.positions_stride + key] : (int)key;
        if (key >= h.length) {
          const uint64_t word = visible ? visible[key - h.length] : (2ull << (key - h.length)) - 1;
          position = start + __popcll(word) - 1;
        }
        position_of[i] = position;
      }
    }
    __syncthreads();
    return c1;
  }
  // key / page by a product (exact for keys below 2^31)
  static __device__ __forceinline__ uint32_t page_index(const TreeParams& p, uint32_t key) { return (uint32_t)(((uint64_t)key * p.page_magic) >> p.page_shift); }
  // the rows of a key, c0: the first key looked up
  template <typename T>
  __device__ __forceinline__ void rows(const TreeParams& p, uint32_t first, uint32_t key, const char*& k, const char*& v) const {
    const uint32_t index = page_index(p, key), slot = key - index * p.cache.page;
    const uint64_t* at = page_at[index - first];
    k = (const char*)(at[0] + slot * (uint64_t)(p.cache.k_slot * (int64_t)sizeof(T)));
    v = (const char*)(at[1] + slot * (uint64_t)(p.cache.v_slot * (int64_t)sizeof(T)));
  }
};

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
      score_at = ((int64_t)head * p.group * p.counted_nodes + hg * p.counted_nodes + __popcll(p.counted & ((1ull << node) - 1))) * (int64_t)p.score_stride;
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

// Of keys k0 .. k0 + 63 the slots of unseen nodes.
__device__ __forceinline__ uint64_t unseen_slots(uint64_t unseen, uint32_t length, uint32_t k0) {
  if (k0 >= length + 64) return ~0ull;
  return k0 >= length ? unseen >> (k0 - length) | ~(~0ull >> (k0 - length)) : length - k0 < 64 ? unseen << (length - k0) : 0;
}

// Four outputs of a row and the logarithm of its sum (base 2): where a run has all of a head's keys to the end, else to the run's
// partial results (slot 0: of the head that it began in the middle of, 1: of the one that it left there).
struct TreePlace {
  const TreeParams& p;
  const TreeHead& h;
  bool all;
  size_t slot;
  __device__ __forceinline__ TreePlace(const TreeParams& p, const TreeHead& h, uint32_t run, uint32_t from, uint32_t to)
      : p(p), h(h), all(from == h.begin && to == h.end), slot((2 * (size_t)run + (from == h.begin ? 1 : 0)) * p.rows) {
    if (threadIdx.x == 0 && p.head_runs) {
      if (from == h.begin) p.head_runs[2 * h.head] = (int)run;
      if (to == h.end) p.head_runs[2 * h.head + 1] = (int)run;
    }
  }
  template <typename T>
  __device__ __forceinline__ void give(uint32_t row, uint32_t column, f32x4 o, float lse) const {
    if (!all) {
      if (column == 0) p.partial_lse[slot + row] = lse;
      store4(p.partial_o + (slot + row) * p.d + column, o);
      return;
    }
    const uint32_t hg = row / p.nodes, node = row - hg * p.nodes, hq = h.hkv * p.group + hg;
    store4((T*)p.o.data + h.batch * p.o.sb + hq * p.o.sh + node * p.o.sn + column, o);
    if (column != 0) return;
    if (p.head_lse) p.head_lse[(size_t)h.head * p.rows + row] = lse;
    if (p.lse) p.lse[((size_t)h.batch * p.hq + hq) * p.nodes + node] = lse * 0.69314718056f;
  }
};

template <typename T, int DPAD, int DUSE, int NW, int RT>
__device__ __forceinline__ void tree_body(const TreeParams& p) {
  using L = Tile<T, DPAD, 32>;
  constexpr int THREADS = 64 * NW, LOADS = 2 * L::WL;
  static_assert(NW >= 2 && 16 * RT <= 32, "nodes in a wavefront's last tile alone");
  static_assert(16 * RT * DPAD * 4 <= 4 * L::BYTES, "a wavefront's result fits its tiles");
  __shared__ __attribute__((aligned(1024))) char smem[NW][2][2][L::BYTES];  // [wavefront][buffer][K, V]
  __shared__ __attribute__((aligned(16))) TreeLookup lookup;
  __shared__ Merge<NW, RT> shared;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t run = blockIdx.x;
  TreeHead head;
  uint32_t unit, stop;
  if (!tree_run(p, run, head, unit, stop)) return;

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[wave][0][0][0]), chunks = p.d * sizeof(T) / 16;
  for (;; head.next(p)) {
    const uint32_t from = unit, to = min(stop, head.end);
    uint32_t c0 = (from - head.begin) * p.unit;
    const uint32_t c2 = min((to - head.begin) * p.unit, head.total);
    const int start = p.start ? p.start[head.batch] : (int)head.length;
    // (the results of the head before lie in the tiles too, where columns past d are to read as zero)
    if (DUSE < DPAD || p.d < DUSE) {
      __syncthreads();
      clear_tiles<NW * 4 * L::BYTES, THREADS>(&smem[0][0][0][0], tid);
    }
    Rows<T, DPAD, DUSE, RT> rows;
    rows.clear();
    TreeRow of[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
      of[b].set(p, head.batch, head.head, head.hkv, 16 * b + r, start);
      rows.load_q(b, of[b].template q<T>(p, head.batch), true, p.d, g);
    }
#pragma unroll
    for (int b = 0; b < RT; ++b) arrive(rows.q[b]);
    while (c0 < c2) {
      const uint32_t c1 = lookup.template fill<T, THREADS>(p, head, start, c0, c2), first = TreeLookup::page_index(p, c0);
      auto request = [&](uint32_t k0, int buf) {
        const char *k[L::WL], *v[L::WL];
#pragma unroll
        for (int w = 0; w < L::WL; ++w) lookup.template rows<T>(p, first, min(k0 + w * L::RPW + lane / L::CH, c1 - 1), k[w], v[w]);
#pragma unroll
        for (int w = 0; w < L::WL; ++w) {
          const uint32_t chunk = (lane % L::CH) ^ L::swizzle(w * L::RPW + lane / L::CH);
          // (a wave-load holds whole rows, so some lane always takes part and the count of transfers in flight is known)
          if (chunk < chunks) {
            dma16_at(k[w] + 16 * chunk, lds + (2 * buf) * L::BYTES + 1024 * w);
            dma16_at(v[w] + 16 * chunk, lds + (2 * buf + 1) * L::BYTES + 1024 * w);
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
            // (32 nodes reach into two tiles at most, the last ones of two wavefronts)
            if (k0 + 32 > head.length && lookup.unseen) clear_rows<L, 1>(&smem[wave][buf][1][0], unseen_slots(lookup.unseen, head.length, k0), 0);
          }
          const bool whole = k0 + 32 <= min(head.length, c1);
          rows.template tile<2>(&smem[wave][buf][0][0], &smem[wave][buf][1][0], bend, whole && !p.slopes && !p.scores, [&](f32x4 (&x)[RT][2]) {
            finish_scores<RT, 2>(p, x, of, lookup.position_of, k0, c0, c1, head.length, whole, g);
          }, reader);
        }
      }
      c0 = c1;
    }
    const TreePlace place(p, head, run, from, to);
    merge_rows(rows, shared, &smem[0][0][0][0], 4 * L::BYTES, p.d, min(16u * RT, p.rows), [&](uint32_t n, uint32_t column, f32x4 o, float lse) {
      place.template give<T>(n, column, o, lse);
    });
    unit = to;
    if (unit == stop) return;
    __syncthreads();  // (the tiles are read)
  }
}

// The same for more rows: up to 64 RT a workgroup, dealt out evenly to its four wavefronts, all of them on the same tile of BN keys; a
// barrier a tile.
template <typename T, int DPAD, int DUSE, int BN, int RT>
__device__ __forceinline__ void tree_rows_body(const TreeParams& p) {
  using L = Tile<T, DPAD, BN>;
  constexpr int NW = 4, KT = BN / 16, EACH = (L::WL + NW - 1) / NW;
  static_assert(L::WL % NW == 0, "tile shape");
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ __attribute__((aligned(16))) TreeLookup lookup;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  // the row tiles of a run on one XCD
  const uint32_t eight = blockIdx.x / 8, row_tile = eight % p.row_tiles, run = eight / p.row_tiles * 8 + blockIdx.x % 8;
  TreeHead head;
  uint32_t unit, stop;
  if (!tree_run(p, run, head, unit, stop)) return;
  // blocks of 16 RT rows: of the row tile, and this wavefront's
  const uint32_t row_blocks = (p.rows + 16 * RT - 1) / (16 * RT), each = (row_blocks + p.row_tiles - 1) / p.row_tiles;
  const uint32_t row_block = row_tile * each + wave, row0 = row_block * (16 * RT);
  const bool active = wave < (int)each && row_block < row_blocks;
  if (DUSE < DPAD || p.d < DUSE) clear_tiles<4 * L::BYTES, 64 * NW>(&smem[0][0][0], tid);

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  const uint32_t lds = lds_address(&smem[0][0][0]), chunks = p.d * sizeof(T) / 16;
  int buf = 0;
  for (;; head.next(p)) {
    const uint32_t from = unit, to = min(stop, head.end);
    uint32_t c0 = (from - head.begin) * p.unit;
    const uint32_t c2 = min((to - head.begin) * p.unit, head.total);
    const int start = p.start ? p.start[head.batch] : (int)head.length;
    Rows<T, DPAD, DUSE, RT> rows;
    rows.clear();
    TreeRow of[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
      of[b].set(p, head.batch, head.head, head.hkv, row0 + 16 * b + r, start);
      rows.load_q(b, of[b].template q<T>(p, head.batch), true, p.d, g);
    }
#pragma unroll
    for (int b = 0; b < RT; ++b) arrive(rows.q[b]);
    while (c0 < c2) {
      const uint32_t c1 = lookup.template fill<T, 64 * NW>(p, head, start, c0, c2), first = TreeLookup::page_index(p, c0);
      auto request = [&](uint32_t k0, int buf) {
        const char *k[EACH], *v[EACH];
#pragma unroll
        for (int it = 0; it < EACH; ++it) lookup.template rows<T>(p, first, min(k0 + (wave + NW * it) * L::RPW + lane / L::CH, c1 - 1), k[it], v[it]);
#pragma unroll
        for (int it = 0; it < EACH; ++it) {
          const uint32_t w = wave + NW * it, chunk = (lane % L::CH) ^ L::swizzle(w * L::RPW + lane / L::CH);
          if (chunk < chunks) {
            dma16_at(k[it] + 16 * chunk, lds + (2 * buf) * L::BYTES + 1024 * w);
            dma16_at(v[it] + 16 * chunk, lds + (2 * buf + 1) * L::BYTES + 1024 * w);
          }
        }
      };
      request(c0, buf);
      for (uint32_t k0 = c0; k0 < c1; k0 += BN, buf ^= 1) {
        dma_wait_all();
        __syncthreads();
        if (k0 + BN < c1) request(k0 + BN, buf ^ 1);
        const bool whole = k0 + BN <= min(head.length, c1);
        if (!whole && lookup.unseen) {
          clear_rows<L, NW>(&smem[buf][1][0], unseen_slots(lookup.unseen, head.length, k0), wave);
          __syncthreads();
        }
        if (!active) continue;
        rows.template tile<KT>(&smem[buf][0][0], &smem[buf][1][0], bend, whole && !p.slopes && !p.scores, [&](f32x4 (&x)[RT][KT]) {
          finish_scores<RT, KT>(p, x, of, lookup.position_of, k0, c0, c1, head.length, whole, g);
        }, reader);
      }
      c0 = c1;
    }
    const TreePlace place(p, head, run, from, to);
#pragma unroll
    for (int b = 0; b < RT; ++b) {
      const float sum = groups_sum(rows.l[b]);
      const uint32_t row = row0 + 16 * b + r;
      if (!active || row >= p.rows) continue;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, lse = rows.m[b] == -INFINITY ? -INFINITY : rows.m[b] + __builtin_amdgcn_logf(sum);
#pragma unroll
      for (int t = 0; t < DUSE / 16; ++t)
        if (16 * t + 4 * g < p.d) place.template give<T>(row, 16 * t + 4 * g, rows.o[b][t] * inv, lse);
    }
    unit = to;
    if (unit == stop) return;
  }
}

// The runs' results of a head put together in their order (a wavefront per row; a head that one run had all of is done already), then
// the weights of the keys: exp(score - lse) over the counted rows, 1024 keys of a head a workgroup.
struct TreeJoin {
  const TreeParams& p;
  uint32_t first, count;  // runs of the head
  __device__ __forceinline__ TreeJoin(const TreeParams& p, uint32_t head)
      : p(p), first((uint32_t)p.head_runs[2 * head]), count((uint32_t)p.head_runs[2 * head + 1] - first + 1) {}
  __device__ __forceinline__ size_t at(uint32_t n, uint32_t row) const { return (2 * (size_t)(first + n) + (n == 0 ? 1 : 0)) * p.rows + row; }
};

template <typename T>
__device__ __forceinline__ void tree_join_body(const TreeParams& p) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t join_blocks = p.whole_heads ? 0 : (p.b * p.hkv * p.rows + 3) / 4;
  if (blockIdx.x < join_blocks) {
    const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + tid / 64));
    if (id >= p.b * p.hkv * p.rows) return;
    const uint32_t head = id / p.rows, row = id - head * p.rows, batch = head / p.hkv, hkv = head - batch * p.hkv;
    const TreeJoin join(p, head);
    if (join.count < 2) return;
    float top = -INFINITY;
    for (uint32_t s = lane; s < join.count; s += 64) top = fmaxf(top, p.partial_lse[join.at(s, row)]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
    for (uint32_t s0 = 0; s0 < join.count; s0 += 64) {
      const float mine = s0 + lane < join.count ? fast_exp2(p.partial_lse[join.at(s0 + lane, row)] - ref) : 0.0f;
      sum += mine;
      const uint32_t here = min(join.count - s0, 64u);
      for (uint32_t s = 0; s < here; ++s) {
        const float weigh = __shfl(mine, (int)s);
        if (4 * lane < p.d) o += *reinterpret_cast<const f32x4*>(p.partial_o + join.at(s0 + s, row) * p.d + 4 * lane) * weigh;
      }
    }
    sum = wave_sum(sum);
    const uint32_t hg = row / p.nodes, node = row - hg * p.nodes, hq = hkv * p.group + hg;
    if (4 * lane < p.d) store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + 4 * lane, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (lane == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = top == -INFINITY ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
    return;
  }
  __shared__ float shared_lse[256];
  const uint32_t tiles = (p.max_length + 1023) / 1024, at = blockIdx.x - join_blocks;
  const uint32_t head = at / tiles, tile = at - head * tiles, batch = head / p.hkv;
  if (head >= p.b * p.hkv) return;
  uint32_t length, total;
  tree_lengths(p, batch, length, total);
  const uint32_t counted = p.group * p.counted_nodes;
  float sum[4] = {0, 0, 0, 0}, before[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t key = 1024 * tile + 256 * k + tid;
    before[k] = key < p.max_length ? p.weights_in[(int64_t)head * p.weights_in_stride + key] : 0.0f;
  }
  if (counted > 0 && 1024 * tile < total) {
    const float* scores = p.scores + (int64_t)head * counted * (int64_t)p.score_stride + 1024 * tile + tid;
    auto score = [&](uint32_t n, int k) { return 1024 * tile + 256 * k + tid < total ? scores[(int64_t)n * (int64_t)p.score_stride + 256 * k] : -INFINITY; };
    // the first rows are under way while the sums of the rows are looked up
    constexpr uint32_t AHEAD = 4;
    float kept[AHEAD][4];
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) kept[n][k] = n < counted ? score(n, k) : -INFINITY;
    const TreeJoin join(p, head);
    for (uint32_t first = 0; first < counted; first += 256) {
      __syncthreads();
      if (first + tid < counted) {
        // counted row n: head n / counted_nodes of the group, the (n % counted_nodes)-th of the counted nodes
        const uint32_t n = first + tid, hg = n / p.counted_nodes;
        uint64_t left = p.counted;
        for (uint32_t k = n - hg * p.counted_nodes; k > 0; --k) left &= left - 1;
        const uint32_t row = hg * p.nodes + __builtin_ctzll(left);
        float lse = 0.0f;
        if (join.count == 1) {
          lse = p.head_lse[(size_t)head * p.rows + row];
        } else {
          float top = -INFINITY, all = 0.0f;
#pragma unroll 4
          for (uint32_t s = 0; s < join.count; ++s) top = fmaxf(top, p.partial_lse[join.at(s, row)]);
          const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
          for (uint32_t s = 0; s < join.count; ++s) all += fast_exp2(p.partial_lse[join.at(s, row)] - ref);
          lse = top == -INFINITY ? -INFINITY : top + __builtin_amdgcn_logf(all);
        }
        shared_lse[tid] = lse == -INFINITY ? INFINITY : lse;
      }
      __syncthreads();
      const uint32_t here = min(counted - first, 256u);
      if (first == 0) {
#pragma unroll
        for (uint32_t n = 0; n < AHEAD; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n < here) sum[k] += fast_exp2(kept[n][k] - shared_lse[n]);
      }
#pragma unroll 4
      for (uint32_t n = first == 0 ? AHEAD : 0; n < here; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += fast_exp2(score(first + n, k) - shared_lse[n]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t key = 1024 * tile + 256 * k + tid;
    if (key < p.max_length) p.weights_out[(int64_t)head * p.weights_out_stride + key] = before[k] + sum[k];
  }
}

}  // namespace attend
