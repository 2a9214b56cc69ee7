// Attention of a few query rows (the nodes of a tree of drafted tokens, or one token) against a long cache in 8 or 4 bits (quantised.h).
//
// Masks, positions, the dealing out of the keys in equal runs and the joining of runs are those of attend_tree.h.  Codes times scales are
// exact in bf16, so that the products are those of a bf16 cache.
#pragma once
#include "quantised.h"

namespace attend {

// Pages of keys c0 ..., by number.
struct QuantisedLookup : TreePositions {
  uint32_t page_at[kTreePages];

  template <int THREADS>
  __device__ __forceinline__ uint32_t fill(const TreeParams& p, const TreeHead& h, int start, uint32_t c0, uint32_t c1) {
    const uint32_t first = page_index(p, c0);
    c1 = end(p, c0, c1);
    const uint32_t pages = page_index(p, c1 - 1) - first + 1;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < pages; i += THREADS) page_at[i] = page_of(p.cache, h.batch, first + i);
    TreePositions::fill<THREADS>(p, h, start, c0, c1);
    __syncthreads();
    return c1;
  }
  // page and slot of a key
  __device__ __forceinline__ void find(const TreeParams& p, uint32_t first, uint32_t key, uint32_t& page, uint32_t& slot) const {
    const uint32_t index = page_index(p, key);
    slot = key - index * p.cache.page;
    page = page_at[index - first];
  }
};

// Rows up to 64 RT a workgroup, dealt out evenly to its four wavefronts, all of them on the same tile of BN keys.  A tile's codes are on
// their way in registers while the tile before is worked on, and reach LDS as bf16 (f32 queries: f32) rows.
template <typename T, int BITS, int DPAD, int BN, int RT>
__device__ __forceinline__ void quantised_rows_body(const QuantisedTreeParams& params) {
  using L = Tile<T, DPAD, BN>;
  using F = Format<BITS>;
  constexpr int NW = 4, KT = BN / 16, BLOCKS = DPAD / 32, PIECES = 2 * BN * BLOCKS, EACH = (PIECES + 64 * NW - 1) / (64 * NW);
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ __attribute__((aligned(16))) QuantisedLookup lookup;
  const TreeParams& p = params.tree;

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
  const uint32_t blocks = (p.d + 31) / 32;
  if (blocks < BLOCKS) clear_tiles<4 * L::BYTES, 64 * NW>(&smem[0][0][0], tid);

  const Bend bend(p.scale, p.cap, p.slopes != nullptr);
  const Reader<T, DPAD> reader(lane);
  int buf = 0;
  for (;; head.next(p)) {
    const uint32_t from = unit, to = min(stop, head.end);
    uint32_t c0 = (from - head.begin) * p.unit;
    const uint32_t c2 = min((to - head.begin) * p.unit, head.total);
    const int start = p.start ? p.start[head.batch] : (int)head.length;
    Rows<T, DPAD, DPAD, RT> rows;
    rows.clear();
    TreeRow of[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
      of[b].set(p, head.batch, head.head, head.hkv, row0 + 16 * b + r, start);
      rows.load_q(b, of[b].template q<T>(p, head.batch), true, p.d, g);
    }
    while (c0 < c2) {
      const uint32_t c1 = lookup.template fill<64 * NW>(p, head, start, c0, c2), first = TreePositions::page_index(p, c0);
      u32x4 codes[EACH][F::BYTES / 16];
      uint32_t bytes[EACH];
      // a piece: a block of a key's row, of K or of V
      auto each_piece = [&](auto use) {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
          const uint32_t i = tid + 64 * NW * n, side = i / (BN * BLOCKS), inside = i % (BN * BLOCKS), key = inside / BLOCKS, block = inside % BLOCKS;
          if (i < PIECES && block < blocks) use(n, side, key, block);
        }
      };
      auto fetch = [&](uint32_t k0) {
        each_piece([&](int n, uint32_t side, uint32_t key, uint32_t block) {
          uint32_t page, slot;
          lookup.find(p, first, min(k0 + key, c1 - 1), page, slot);
          const QuantisedSide& s = side ? params.v : params.k;
          const uint8_t* at = s.codes + (int64_t)page * s.page + (int64_t)head.hkv * s.head + (int64_t)slot * s.slot + block * F::BYTES;
#pragma unroll
          for (int w = 0; w < F::BYTES / 16; ++w) codes[n][w] = ldg128(at + 16 * w);
          bytes[n] = (s.scales + (int64_t)page * s.scale_page + (int64_t)head.hkv * s.scale_head + (int64_t)slot * s.scale_slot)[block];
        });
      };
      auto write = [&](int buf) {
        each_piece([&](int n, uint32_t side, uint32_t key, uint32_t block) {
          char* row = &smem[buf][side][0] + key * L::RB;
          const float scale = scale_of(bytes[n]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t words[BITS / 4];
#pragma unroll
            for (int w = 0; w < BITS / 4; ++w) words[w] = codes[n][(c * (BITS / 4) + w) / 4][(c * (BITS / 4) + w) % 4];
            const Frag<T> x = decode<BITS>(words, scale, T());
            constexpr int CHUNKS = (int)sizeof(T) / 2;  // 16-byte chunks of 8 columns
#pragma unroll
            for (int h = 0; h < CHUNKS; ++h) {
              const uint32_t chunk = (CHUNKS * (4 * block + c) + h) ^ L::swizzle(key);
              if constexpr (CHUNKS == 1) *reinterpret_cast<Frag<T>*>(row + 16 * chunk) = x;
              else *reinterpret_cast<f32x4*>(row + 16 * chunk) = f32x4{x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
            }
          }
        });
      };
      fetch(c0);
      for (uint32_t k0 = c0; k0 < c1; k0 += BN, buf ^= 1) {
        write(buf);  // (the other buffer may still be read)
        __syncthreads();
        if (k0 + BN < c1) fetch(k0 + BN);
        const bool whole = k0 + BN <= min(head.length, c1);
        if (!whole && lookup.unseen) {
          clear_rows<L, NW>(&smem[buf][1][0], unseen_slots(lookup.unseen, head.length, k0), wave);
          __syncthreads();
        }
        if (!active) continue;
        rows.template tile<KT>(&smem[buf][0][0], &smem[buf][1][0], bend, whole && !p.slopes, [&](f32x4 (&x)[RT][KT]) {
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
      for (int t = 0; t < DPAD / 16; ++t)
        if (16 * t + 4 * g < p.d) place.template give<T>(row, 16 * t + 4 * g, rows.o[b][t] * inv, lse);
    }
    unit = to;
    if (unit == stop) return;
  }
}

}  // namespace attend
