// Attention of a few query rows (the nodes of a tree of drafted tokens, or one token) against a long cache in 8 or 4 bits (quantised.h).
//
// Masks, positions, the dealing out of the keys in equal runs and the joining of runs are those of attend_tree.h.  Codes times scales are
// exact in bf16, so that the products are those of a bf16 cache.
#pragma once
#include "quantised.h"

namespace attend {

// Pages of keys c0 ..., by number.  What a look-up needs is requested from memory in one step, and taken over in another.
struct QuantisedLookup : TreePositions {
  uint32_t page_at[kTreePages];

  template <int THREADS>
  struct Request {
    uint32_t first, c0, c1, page[kTreePages / THREADS];
    uint64_t seen;  // by a node of this lane
    // keys c0 .. c2 - 1, as many as there is room for
    __device__ __forceinline__ void operator()(const TreeParams& p, const TreeHead& h, uint32_t from, uint32_t c2) {
      c0 = from;
      first = page_index(p, c0);
      c1 = end(p, c0, c2);
      const uint32_t last = page_index(p, c1 - 1);
#pragma unroll
      for (int n = 0; n < kTreePages / THREADS; ++n) page[n] = page_of(p.cache, h.batch, min(first + threadIdx.x + THREADS * n, last));
      seen = p.visible ? p.visible[(int64_t)h.batch * p.visible_stride + min((uint32_t)lane_now(), p.nodes - 1)] : 0;
    }
  };
  // by all threads, between two barriers
  template <int THREADS>
  __device__ __forceinline__ void take(const TreeParams& p, const TreeHead& h, int start, const Request<THREADS>& request) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kTreePages / THREADS; ++n) page_at[threadIdx.x + THREADS * n] = request.page[n];
    if (threadIdx.x < 64) {
      const uint64_t nodes = unseen_of(p, request.seen);
      if (threadIdx.x == 0) unseen = nodes;
    }
    fill_positions<THREADS>(p, h, start, request.c0, request.c1);
    __syncthreads();
  }
  // page and slot of a key
  __device__ __forceinline__ void find(const TreeParams& p, uint32_t first, uint32_t key, uint32_t& page, uint32_t& slot) const {
    const uint32_t index = page_index(p, key);
    slot = key - index * p.cache.page;
    page = page_at[index - first];
  }
};

// The kernel's arguments, read anew.  There are more of them than scalar registers: left to itself the compiler reads them all at the
// start and keeps what does not fit in lanes of vector registers (127 moves there before the first tile, and back).
__device__ __forceinline__ const QuantisedTreeParams& arguments() {
  auto at = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const QuantisedTreeParams*)at;
}

// A pointer that is known to point to memory, not to LDS (one that comes from an address, or from an argument read anew, is not: loads
// through it would count as reads of LDS too).
template <typename T>
using Memory = const __attribute__((address_space(1))) T*;
__device__ __forceinline__ u32x4 ldg128(Memory<uint8_t> at) { return *(Memory<u32x4>)at; }

// Products of f32 queries and probabilities with what codes stand for, which is exact in bf16: in three bf16 parts, which hold their 24
// bits, on the bf16 matrix instructions (three take 48 cycles where the eight f32 ones take 256).  bf16: one part, the nearest, as over a
// bf16 cache: probabilities are off by up to 2^-8 of themselves, which a second part, and with it a second product with V, would save (o is 2.3e-3 from 64
// bits, 1.7e-3 of that its own rounding).
template <int PARTS, int N>
__device__ __forceinline__ void into_parts(const float (&x)[N], bf16_t (&part)[PARTS][N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float left = x[e];
#pragma unroll
    for (int n = 0; n < PARTS; ++n) {
      part[n][e] = (bf16_t)left;
      left -= (float)part[n][e];
    }
  }
}

// 16 query rows of a wavefront in parts, and their running softmax (that of Rows).
template <typename T, int DPAD, int KT>
struct PartRows {
  static constexpr int PARTS = std::is_same_v<T, float> ? 3 : 1, KS = DPAD / 32;
  Rows<bf16_t, DPAD, DPAD, 1> rows;  // (its queries: the first part)
  bf16x8 more[PARTS][KS];            // the other parts
  // operand ks: columns first + step ks .. + 7
  __device__ __forceinline__ void load_q(Memory<T> row, uint32_t d, uint32_t first, uint32_t step) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t at = first + step * ks;
      Frag<T> x = zero_frag<T>();
      if (at < d) x = *(Memory<Frag<T>>)(row + at);
      if constexpr (PARTS == 1) {
        rows.q[0][ks] = x;
      } else {
        float y[8];
        bf16_t part[PARTS][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e];
        into_parts(y, part);
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
          bf16x8& to = n == 0 ? rows.q[0][ks] : more[n - 1][ks];
#pragma unroll
          for (int e = 0; e < 8; ++e) to[e] = part[n][e];
        }
      }
    }
  }
  __device__ __forceinline__ f32x4 product(bf16x8 a, int ks, f32x4 sum) const {
    sum = mma(a, rows.q[0][ks], sum);
#pragma unroll
    for (int n = 1; n < PARTS; ++n) sum = mma(a, more[n - 1][ks], sum);
    return sum;
  }
  template <typename Exponent>
  __device__ __forceinline__ bool weigh(const f32x4 (&s)[1][KT], Exponent exponent, f32x4 (&e)[KT], float& sum) const {
    const float ref = rows.m[0] == -INFINITY ? 0.0f : rows.m[0];
    float part[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[t][i] = fast_exp2(exponent(s[0][t][i], ref));
        part[i & 1] += e[t][i];
      }
    sum = part[0] + part[1];
    return __builtin_amdgcn_ballot_w64(!(sum < 0x1p30f && rows.m[0] > -INFINITY)) == 0;
  }
  // products into probabilities (as Rows::tile, but for the products, which are kept instead of computed again)
  template <typename Finish>
  __device__ __forceinline__ void probabilities(f32x4 (&s)[1][KT], const Bend& bend, bool plain, Finish finish, f32x4 (&e)[KT]) {
    float sum;
    bool done = false;
    if (plain) {
      if (!bend.bent) done = weigh(s, [&](float x, float ref) { return __builtin_fmaf(x, bend.mult, -ref); }, e, sum);
      else if (bend.capped && bend.all_small(s)) done = weigh(s, [&](float x, float ref) { return __builtin_fmaf(x, bend.small(x * x), -ref); }, e, sum);
    }
    if (!done) {
      if (bend.bent) {
        bend.all(s);
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) s[0][t] *= bend.mult;
      }
      finish(s);
      rows.move(s);
      weigh(s, [](float x, float ref) { return x - ref; }, e, sum);
    }
    rows.l[0] += sum;
  }
};

// ---- more rows ------------------------------------------------------------------------------------------------------------
//
// 64 rows a workgroup, 16 for each of its four wavefronts, all of them on the same tile of BN keys.  A tile's codes are on their way in
// registers while the tile before is worked on, and reach LDS as bf16 rows, decoded once for all rows.
// 32 rows a wavefront would share its operand reads, but leave room for two wavefronts a SIMD instead of three: 8 x 8 heads of 4096 x
// 128 at 4 bits, 4 query heads a key head, us a call with 16 and 32 rows: 12 nodes 28 and 32, 24 nodes 38 and 40, 48 nodes 48 and 51, 64
// nodes 57 and 58;  32 x 8 heads of 8192, 16 nodes 85 and 110.
template <typename T, int BITS, int DPAD, int BN>
__device__ __forceinline__ void quantised_rows_body(const QuantisedTreeParams& params) {
  using L = Tile<bf16_t, DPAD, BN>;
  using F = Format<BITS>;
  constexpr int NW = 4, THREADS = 64 * NW, KT = BN / 16, BLOCKS = DPAD / 32, PIECES = 2 * BN * BLOCKS, EACH = (PIECES + THREADS - 1) / THREADS;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][L::BYTES];  // [buffer][K, V]
  __shared__ __attribute__((aligned(16))) QuantisedLookup lookup;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  // the row tiles of a run on one XCD
  const uint32_t eight = blockIdx.x / 8, row_tiles = params.tree.row_tiles, row_tile = eight % row_tiles, run = eight / row_tiles * 8 + blockIdx.x % 8;
  TreeHead head;
  uint32_t unit, stop;
  if (!tree_run(arguments().tree, run, head, unit, stop)) return;
  unit = max(unit, head.begin);
  if (unit >= stop) return;
  // blocks of 16 rows: of the row tile, and this wavefront's
  const uint32_t row_blocks = (params.tree.rows + 15) / 16, each = (row_blocks + row_tiles - 1) / row_tiles;
  const uint32_t row_block = row_tile * each + wave, row0 = row_block * 16;
  const bool active = wave < (int)each && row_block < row_blocks;
  const uint32_t blocks = (params.tree.d + 31) / 32;
  if (blocks < BLOCKS) clear_tiles<4 * L::BYTES, THREADS>(&smem[0][0][0], tid);

  const bool biased = params.tree.slopes != nullptr;
  const Bend bend(params.tree.scale, params.tree.cap, biased);
  const Reader<bf16_t, DPAD> reader(lane);
  int buf = 0;
  // (requests as in quantised_few_body)
  uint32_t from, to, c0, c2;
  int start;
  PartRows<T, DPAD, KT> part_rows;
  auto& rows = part_rows.rows;
  TreeRow of[1];
  QuantisedLookup::Request<THREADS> request;
  auto begin = [&](const TreeHead& h) {
    const TreeParams& p = arguments().tree;
    from = unit;
    to = min(stop, h.end);
    c0 = (from - h.begin) * p.unit;
    c2 = min((to - h.begin) * p.unit, h.total);
    start = p.start ? p.start[h.batch] : (int)h.length;
    request(p, h, c0, c2);
    of[0].set(p, h.batch, h.head, h.hkv, row0 + r, start);
    part_rows.load_q((Memory<T>)of[0].template q<T>(p, h.batch), p.d, 8 * g, 32);
  };
  begin(head);
  for (;;) {
    rows.clear();
    for (;;) {
      lookup.take(arguments().tree, head, start, request);
      const uint32_t c1 = request.c1, first = request.first;
      u32x4 codes[EACH][F::BYTES / 16];
      uint32_t bytes[EACH];
      // a piece: a block of a key's row, of K or of V
      auto each_piece = [&](auto use) {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
          const uint32_t i = tid + THREADS * n, side = i / (BN * BLOCKS), inside = i % (BN * BLOCKS), key = inside / BLOCKS, block = inside % BLOCKS;
          if (i < PIECES && block < blocks) use(n, side, key, block);
        }
      };
      auto fetch = [&](uint32_t k0) {
        each_piece([&](int n, uint32_t side, uint32_t key, uint32_t block) {
          uint32_t page, slot;
          lookup.find(params.tree, first, min(k0 + key, c1 - 1), page, slot);
          const QuantisedSide& s = side ? params.v : params.k;
          const Memory<uint8_t> at = (Memory<uint8_t>)(s.codes + (int64_t)page * s.page + (int64_t)head.hkv * s.head + (int64_t)slot * s.slot + block * F::BYTES);
#pragma unroll
          for (int w = 0; w < F::BYTES / 16; ++w) codes[n][w] = ldg128(at + 16 * w);
          bytes[n] = ((Memory<uint8_t>)(s.scales + (int64_t)page * s.scale_page + (int64_t)head.hkv * s.scale_head + (int64_t)slot * s.scale_slot))[block];
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
            *reinterpret_cast<bf16x8*>(row + 16 * ((4 * block + c) ^ L::swizzle(key))) = decode<BITS>(words, scale, bf16_t());
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
        const char *const k_tile = &smem[buf][0][0], *const v_tile = &smem[buf][1][0];
        auto finish = [&](f32x4 (&x)[1][KT]) {
          finish_scores<1, KT>(arguments().tree, x, of, lookup.position_of, k0, c0, c1, head.length, whole, g);
        };
        if constexpr (part_rows.PARTS == 1) {
          rows.template tile<KT>(k_tile, v_tile, bend, whole && !biased, finish, reader);
        } else {
          f32x4 s[1][KT], e[KT];
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            s[0][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < DPAD / 32; ++ks) s[0][t] = part_rows.product(reader.rows(k_tile, t, ks), ks, s[0][t]);
          }
          settle<bf16_t>(s[0]);
          part_rows.probabilities(s, bend, whole && !biased, finish, e);
#pragma unroll
          for (int u = 0; u < KT / 2; ++u) {
            float y[8];
            bf16_t part[part_rows.PARTS][8];
#pragma unroll
            for (int n = 0; n < 8; ++n) y[n] = e[2 * u + n / 4][n % 4];
            into_parts(y, part);
            bf16x8 pf[part_rows.PARTS];
#pragma unroll
            for (int m = 0; m < part_rows.PARTS; ++m)
#pragma unroll
              for (int n = 0; n < 8; ++n) pf[m][n] = part[m][n];
#pragma unroll
            for (int t = 0; t < DPAD / 16; ++t) {
              const bf16x8 a = reader.across(v_tile, t, u);
#pragma unroll
              for (int m = 0; m < part_rows.PARTS; ++m) rows.o[0][t] = mma(a, pf[m], rows.o[0][t]);
            }
          }
        }
      }
      c0 = c1;
      if (c0 == c2) break;
      request(arguments().tree, head, c0, c2);
    }
    const TreeParams& p = arguments().tree;
    const TreeHead done = head;
    const TreePlace place(p, done, run, from, to);
    bool last = to == stop;
    if (!last) {
      head.next(p);
      unit = head.begin;
      last = unit >= stop;
      if (!last) begin(head);
    }
    const float sum = groups_sum(rows.l[0]);
    const uint32_t row = row0 + r;
    if (active && row < p.rows) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, lse = rows.m[0] == -INFINITY ? -INFINITY : rows.m[0] + __builtin_amdgcn_logf(sum);
#pragma unroll
      for (int t = 0; t < DPAD / 16; ++t)
        if (16 * t + 4 * g < p.d) place.template give<T>(row, 16 * t + 4 * g, rows.o[0][t] * inv, lse);
    }
    if (last) return;
  }
}

// ---- up to 16 rows: the step of a token --------------------------------------------------------------------------------------
//
// Every wavefront walks tiles of 16 KT keys of its own, with no barrier.  Codes of the next tile are on their way in registers while a
// tile is worked on, and stay codes as long as they can:
//   K  lane (r, g) of a 16-key block has a quarter of key r's row, the columns DPAD / 4 g ...; 8 of them make an operand.  (Which
//      columns a step adds up does not matter as long as the queries' operand agrees.)  The scale is the conversion's.
//   V  the second product wants 8 keys of a column in a lane.  Codes pass through LDS as they are and are read transposed, 4 bits: 16
//      keys of a column a lane, 8 bits: 8 keys.  Scales differ from key to key then; they are powers of two, so a probability times its
//      key's scale is as exact as the probability, and goes into the product in its place, anew for every 32 columns.
//      (Where values are below 2^-110 such a product may lie below the smallest bf16 and is lost, and its lesser parts (f32) from 2^-80 on.  A
//      probability may reach 2^30 before its reference follows: above 2^97 the product may be infinite.  The outputs are promised for
//      values from 2^-80 to 2^70 in magnitude.)

template <int BITS>
__device__ __forceinline__ constexpr int few_blocks() { return BITS == 4 ? 4 : 2; }  // 16-key blocks of a tile

// Where the 16-byte chunks of V's rows lie: chunk c of key k at c ^ swizzle(k), so that 16 keys read at one chunk (k = 16 run + 4 g + i for
// all run and i) meet no bank twice (rows of 32 bytes: two do).
template <int CH>
__device__ __forceinline__ uint32_t few_swizzle(uint32_t k) {
  if constexpr (CH == 2) return k >> 4 & 1;
  if constexpr (CH == 4) return k >> 4 & 3;
  if constexpr (CH == 8) return (k >> 4 & 3) | (k >> 1 & 1) << 2;
  return (k >> 4 & 3) | (k & 3) << 2;
}

template <int BYTES>
struct Words {
  uint32_t w[BYTES / 4];
  __device__ __forceinline__ void load(Memory<uint8_t> at) {
    if constexpr (BYTES == 8) {
      const u32x2 x = *(Memory<u32x2>)at;
      w[0] = x[0];
      w[1] = x[1];
    } else {
#pragma unroll
      for (int n = 0; n < BYTES / 16; ++n) {
        const u32x4 x = ldg128(at + 16 * n);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * n + e] = x[e];
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < BYTES / 4; ++n) w[n] = 0;
  }
};

// The codes and scales of a tile of a wavefront, on their way.
template <int BITS, int DPAD>
struct FewTile {
  static constexpr int KT = few_blocks<BITS>(), BLOCKS = DPAD / 32;
  static constexpr int KB = DPAD / 4 * BITS / 8;  // bytes of a key's codes that a lane has
  static constexpr int KS = DPAD == 256 ? 2 : 1;  // ... and scales
  static constexpr int RB = DPAD * BITS / 8, CH = RB / 16;
  static constexpr int VL = 16 * KT * RB / 1024;  // 16-byte loads of V a lane
  Words<KB> k[KT];
  uint32_t k_scale[KT][KS];
  u32x4 v[VL];
  uint32_t v_scale[BLOCKS];
};

// Requests of tiles of one key head.  Columns past the row's blocks are read as those of its last block: the queries' operand is zero
// there, and outputs of such columns are not written.
template <int BITS, int DPAD>
struct FewFetch {
  using Tile = FewTile<BITS, DPAD>;
  using F = Format<BITS>;
  static constexpr int KEYS = 16 * Tile::KT;
  const QuantisedTreeParams& params;
  const QuantisedLookup& lookup;
  uint32_t lane;
  uint32_t k_at[Tile::KS], k_scale_at[Tile::KS];  // of this lane in K's rows (a block each)
  uint32_t v_key, v_at[Tile::VL];                 // ... in V's: key in the first load, and bytes of all of them
  uint32_t blocks;
  Memory<uint8_t> k, k_scales, v, v_scales;       // the head's rows of page 0
  __device__ __forceinline__ FewFetch(const QuantisedTreeParams& params, const QuantisedLookup& lookup)
      : params(params), lookup(lookup), lane(threadIdx.x & 63), blocks((params.tree.d + 31) / 32) {
    const uint32_t g = lane >> 4;
#pragma unroll
    for (int n = 0; n < Tile::KS; ++n) {
      const uint32_t block = DPAD == 64 ? g / 2 : DPAD == 128 ? g : 2 * g + n;
      k_scale_at[n] = min(block, blocks - 1);
      k_at[n] = k_scale_at[n] * F::BYTES + (DPAD == 64 ? g % 2 * (F::BYTES / 2) : 0);
    }
    v_key = lane / Tile::CH;
#pragma unroll
    for (int m = 0; m < Tile::VL; ++m) {
      const uint32_t n = 64 * m + lane, chunk = (n % Tile::CH) ^ few_swizzle<Tile::CH>(n / Tile::CH);
      v_at[m] = min(16 * chunk, blocks * F::BYTES - 16);
    }
  }
  __device__ __forceinline__ void of_head(uint32_t hkv) {
    k = (Memory<uint8_t>)(params.k.codes + (int64_t)hkv * params.k.head);
    k_scales = (Memory<uint8_t>)(params.k.scales + (int64_t)hkv * params.k.scale_head);
    v = (Memory<uint8_t>)(params.v.codes + (int64_t)hkv * params.v.head);
    v_scales = (Memory<uint8_t>)(params.v.scales + (int64_t)hkv * params.v.scale_head);
  }
  // Keys k0 .. k0 + KEYS - 1, where one is past c1 - 1 that one instead.
  __device__ __forceinline__ void operator()(Tile& x, uint32_t first, uint32_t k0, uint32_t c1) const {
    const TreeParams& p = params.tree;
    if (p.cache.page % KEYS == 0 && k0 + KEYS <= c1) {
      // all of them in one page: addresses are the wavefront's
      const uint32_t index = TreePositions::page_index(p, k0), slot = k0 - index * p.cache.page;
      const int64_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)lookup.page_at[index - first]);
      const Memory<uint8_t> k_row = k + page * params.k.page + (int64_t)slot * params.k.slot;
      const Memory<uint8_t> k_scale_row = k_scales + page * params.k.scale_page + (int64_t)slot * params.k.scale_slot;
      const Memory<uint8_t> v_row = v + page * params.v.page + (int64_t)slot * params.v.slot;
      const Memory<uint8_t> v_scale_row = v_scales + page * params.v.scale_page + (int64_t)slot * params.v.scale_slot;
      const uint32_t r = lane & 15, k_stride = (uint32_t)params.k.slot, k_scale_stride = (uint32_t)params.k.scale_slot, v_stride = (uint32_t)params.v.slot;
#pragma unroll
      for (int t = 0; t < Tile::KT; ++t) load_k(x, t, k_row + (int64_t)(16 * t) * k_stride, k_scale_row + (int64_t)(16 * t) * k_scale_stride, r * k_stride, r * k_scale_stride);
#pragma unroll
      for (int m = 0; m < Tile::VL; ++m) x.v[m] = ldg128(v_row + (int64_t)(64 / Tile::CH * m) * v_stride + (v_key * v_stride + v_at[m]));
      load_v_scales(x, v_scale_row + lane % KEYS * (uint32_t)params.v.scale_slot);
      return;
    }
    // a lane finds the rows of one key, and hands them to those that need them
    const uint32_t key = min(k0 + lane % KEYS, c1 - 1);
    uint32_t page, slot;
    lookup.find(p, first, key, page, slot);
    const uint64_t k_row = (uint64_t)k + page * (uint64_t)params.k.page + slot * (uint64_t)params.k.slot;
    const uint64_t k_scale_row = (uint64_t)k_scales + page * (uint64_t)params.k.scale_page + slot * (uint64_t)params.k.scale_slot;
    const uint64_t v_row = (uint64_t)v + page * (uint64_t)params.v.page + slot * (uint64_t)params.v.slot;
#pragma unroll
    for (int t = 0; t < Tile::KT; ++t) load_k(x, t, of_lane(k_row, 16 * t + (lane & 15)), of_lane(k_scale_row, 16 * t + (lane & 15)), 0, 0);
#pragma unroll
    for (int m = 0; m < Tile::VL; ++m) x.v[m] = ldg128(of_lane(v_row, 64 / Tile::CH * m + v_key) + v_at[m]);
    load_v_scales(x, (Memory<uint8_t>)((uint64_t)v_scales + page * (uint64_t)params.v.scale_page + slot * (uint64_t)params.v.scale_slot));
  }

 private:
  static __device__ __forceinline__ Memory<uint8_t> of_lane(uint64_t at, uint32_t from) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(4 * from), (int)(uint32_t)at);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(4 * from), (int)(uint32_t)(at >> 32));
    return (Memory<uint8_t>)((uint64_t)hi << 32 | lo);
  }
  __device__ __forceinline__ void load_k(Tile& x, int t, Memory<uint8_t> row, Memory<uint8_t> scale_row, uint32_t at, uint32_t scale_at) const {
    constexpr int WORDS = Tile::KB / 4 / Tile::KS;
#pragma unroll
    for (int n = 0; n < Tile::KS; ++n) {
      x.k_scale[t][n] = scale_row[scale_at + k_scale_at[n]];
      Words<4 * WORDS> part;
      part.load(row + (at + k_at[n]));
#pragma unroll
      for (int w = 0; w < WORDS; ++w) x.k[t].w[WORDS * n + w] = part.w[w];
    }
  }
  __device__ __forceinline__ void load_v_scales(Tile& x, Memory<uint8_t> row) const {
#pragma unroll
    for (uint32_t n = 0; n < Tile::BLOCKS; ++n) x.v_scale[n] = row[min(n, blocks - 1)];
  }
};

typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((address_space(3))) i32x2* lds_i32x2_ptr;

template <typename T, int BITS, int DPAD>
struct FewRows : PartRows<T, DPAD, few_blocks<BITS>()> {
  using Held = FewTile<BITS, DPAD>;
  using Base = PartRows<T, DPAD, few_blocks<BITS>()>;
  using Base::PARTS, Base::KS, Base::rows;
  static constexpr int KT = Held::KT, CH = Held::CH, RB = Held::RB, BLOCKS = Held::BLOCKS;
  static constexpr int V_BYTES = 16 * KT * RB, SCALE_BYTES = BLOCKS * 16 * KT * 4;

  // V's codes and scales to this wavefront's LDS.  `without`: keys whose rows are set to zero.
  static __device__ __forceinline__ void put(const Held& x, char* v, float* scales, int lane, uint64_t without) {
#pragma unroll
    for (int m = 0; m < Held::VL; ++m) *reinterpret_cast<u32x4*>(v + 16 * (64 * m + lane)) = x.v[m];
    const uint32_t key = lane % (16 * KT);  // (32 keys: two lanes write the same)
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) scales[16 * KT * n + key] = scale_of(x.v_scale[n]);
    if (without == 0) return;
#pragma unroll 1
    for (int m = 0; m < Held::VL; ++m)
      if (without >> ((64 * m + lane) / CH) & 1) *reinterpret_cast<u32x4*>(v + 16 * (64 * m + lane)) = u32x4{0, 0, 0, 0};
    if (without >> key & 1) {
#pragma unroll 1
      for (int n = 0; n < BLOCKS; ++n) scales[16 * KT * n + key] = 0.0f;
    }
  }
  // S^T of the tile
  __device__ __forceinline__ void products(const Held& x, f32x4 (&s)[1][KT]) const {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      s[0][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 a = decode<BITS>(&x.k[t].w[BITS / 4 * ks], scale_of(x.k_scale[t][DPAD == 256 ? ks / 4 : 0]), bf16_t());
        s[0][t] = this->product(a, ks, s[0][t]);
      }
    }
    settle<bf16_t>(s[0]);
  }
  template <typename Finish>
  __device__ __forceinline__ void add(f32x4 (&s)[1][KT], const char* v, const float* scales, const Bend& bend, bool plain, Finish finish, int r, int g) {
    f32x4 e[KT];
    this->probabilities(s, bend, plain, finish, e);
    // this lane's place in V: 4 bits: key 16 (j / 4) + 4 g + j % 4, j = r;  8 bits: j = r / 2, half r % 2 of the 16-byte chunk
    const uint32_t j = BITS == 4 ? r : r / 2, key = 16 * (j / 4) + 4 * g + j % 4;
    const char* row = v + key * RB;
    const uint32_t swizzle = few_swizzle<CH>(key);
#pragma unroll
    for (int block = 0; block < BLOCKS; ++block) {
      bf16x8 pf[PARTS][KT / 2];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f32x4 scale = *reinterpret_cast<const f32x4*>(scales + 16 * KT * block + 16 * t + 4 * g);
        float y[4];
        bf16_t part[PARTS][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = e[t][i] * scale[i];
        into_parts(y, part);
#pragma unroll
        for (int n = 0; n < PARTS; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) pf[n][t / 2][4 * (t & 1) + i] = part[n][i];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x4& o = rows.o[0][2 * block + half];
        if constexpr (BITS == 4) {
          // 16 columns: half a chunk
          const i32x2 codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr)(row + 16 * (block ^ swizzle) + 8 * half));
#pragma unroll
          for (int u = 0; u < KT / 2; ++u) {
            const uint32_t word = (uint32_t)codes[u];
            const bf16x8 a = decode<4>(&word, 1.0f, bf16_t());
#pragma unroll
            for (int n = 0; n < PARTS; ++n) o = mma(a, pf[n][u], o);
          }
        } else {
          const i32x2 codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_ptr)(row + 16 * ((2 * block + half) ^ swizzle) + 8 * (r & 1)));
          const uint32_t words[2] = {(uint32_t)codes[0], (uint32_t)codes[1]};
          const bf16x8 a = decode<8>(words, 1.0f, bf16_t());
#pragma unroll
          for (int n = 0; n < PARTS; ++n) o = mma(a, pf[n][0], o);
        }
      }
    }
  }
};

template <typename T, int BITS, int DPAD, int NW>
__device__ __forceinline__ void quantised_few_body(const QuantisedTreeParams& params) {
  using R = FewRows<T, BITS, DPAD>;
  using Held = FewTile<BITS, DPAD>;
  constexpr int THREADS = 64 * NW, KT = R::KT, KEYS = 16 * KT;
  constexpr int USED = R::V_BYTES + R::SCALE_BYTES, RESULT = 16 * DPAD * 4, BYTES = USED > RESULT ? USED : RESULT;
  __shared__ __attribute__((aligned(1024))) char smem[NW][BYTES];
  __shared__ __attribute__((aligned(16))) QuantisedLookup lookup;
  __shared__ Merge<NW, 1> shared;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t run = blockIdx.x;
  TreeHead head;
  uint32_t unit, stop;
  if (!tree_run(arguments().tree, run, head, unit, stop)) return;
  unit = max(unit, head.begin);
  if (unit >= stop) return;

  const bool biased = params.tree.slopes != nullptr;
  const Bend bend(params.tree.scale, params.tree.cap, biased);
  FewFetch<BITS, DPAD> fetch(params, lookup);
  char* const v = &smem[wave][0];
  float* const scales = reinterpret_cast<float*>(v + R::V_BYTES);
  // Of a key head: what its first keys need from memory is all requested at once, that of the next head before the results of the one
  // before are put together.
  uint32_t from, to, c0, c2;
  int start;
  R few;
  TreeRow of[1];
  QuantisedLookup::Request<THREADS> request;
  auto begin = [&](const TreeHead& h) {
    const TreeParams& p = arguments().tree;
    from = unit;
    to = min(stop, h.end);
    c0 = (from - h.begin) * p.unit;
    c2 = min((to - h.begin) * p.unit, h.total);
    start = p.start ? p.start[h.batch] : (int)h.length;
    request(p, h, c0, c2);
    of[0].set(p, h.batch, h.head, h.hkv, r, start);
    few.load_q((Memory<T>)of[0].template q<T>(p, h.batch), p.d, DPAD / 4 * g, 8);
  };
  begin(head);
  for (;;) {
    few.rows.clear();
    fetch.of_head(head.hkv);
    for (;;) {
      lookup.take(arguments().tree, head, start, request);
      const uint32_t c1 = request.c1, first = request.first;
      // (one place that requests a tile, the first one too: the code of it is long)
      Held next;
      for (uint32_t ahead = c0 + KEYS * wave;; ahead += KEYS * NW) {
        const uint32_t k0 = ahead - KEYS * NW;  // the tile that has arrived, if this is not the first request
        const bool begun = ahead >= c0 + KEYS * NW, more = ahead < c1;
        if (!begun && !more) break;
        const bool whole = k0 + KEYS <= min(head.length, c1);
        const Held held = next;
        if (begun) {
          const uint64_t without = !whole && lookup.unseen ? unseen_slots(lookup.unseen, head.length, k0) : 0;
          asm volatile("" ::: "memory");
          R::put(held, v, scales, lane, without);
          asm volatile("" ::: "memory");
        }
        if (more) fetch(next, first, ahead, c1);
        if (!begun) continue;
        f32x4 s[1][KT];
        few.products(held, s);
        few.add(s, v, scales, bend, whole && !biased, [&](f32x4 (&x)[1][KT]) {
          finish_scores<1, KT>(arguments().tree, x, of, lookup.position_of, k0, c0, c1, head.length, whole, g);
        }, r, g);
        if (!more) break;
      }
      c0 = c1;
      if (c0 == c2) break;
      request(arguments().tree, head, c0, c2);
    }
    const TreeParams& p = arguments().tree;
    const TreeHead done = head;
    const TreePlace place(p, done, run, from, to);
    bool last = to == stop;
    if (!last) {
      head.next(p);
      unit = head.begin;
      last = unit >= stop;
      if (!last) begin(head);
    }
    merge_rows(few.rows, shared, &smem[0][0], BYTES, p.d, p.rows, [&](uint32_t n, uint32_t column, f32x4 o, float lse) {
      place.template give<T>(n, column, o, lse);
    });
    if (last) return;
  }
}

// The runs' results of a row put together: as many lanes a row as have four columns each, eight runs at a time, whose sums' logarithms and
// results are all on their way at once (every lane computes the runs' weights itself).  (A wavefront a row and one run after the other, as
// attend_tree_join has it: 12288 rows of four to six runs 11.0 us; this 7.4.)
template <typename T, int DPAD>
__device__ __forceinline__ void quantised_few_join_body(const TreeParams& p) {
  constexpr uint32_t COLUMNS = DPAD / 4, AHEAD = 8;
  const uint32_t id = blockIdx.x * (256 / COLUMNS) + threadIdx.x / COLUMNS, column = 4 * (threadIdx.x % COLUMNS);
  if (id >= p.b * p.hkv * p.rows) return;
  const uint32_t head = id / p.rows, row = id - head * p.rows, batch = head / p.hkv, hkv = head - batch * p.hkv;
  const TreeJoin join(p, head);
  if (join.count < 2) return;
  float top = -INFINITY, sum = 0.0f;
  f32x4 o = {0, 0, 0, 0};
  for (uint32_t s0 = 0; s0 < join.count; s0 += AHEAD) {
    float lse[AHEAD];
    f32x4 part[AHEAD];
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) {
      lse[n] = -INFINITY;
      part[n] = f32x4{0, 0, 0, 0};
      if (s0 + n >= join.count) continue;
      const size_t at = join.at(s0 + n, row);
      lse[n] = p.partial_lse[at];
      if (column < p.d) part[n] = *reinterpret_cast<const f32x4*>(p.partial_o + at * p.d + column);
    }
    float above = top;
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) above = fmaxf(above, lse[n]);
    // (a score that is no number makes its row one: the maximum passes it over)
    const float ref = above == -INFINITY ? 0.0f : above, before = fast_exp2(top - ref);
    top = above;
    sum *= before;
    o *= before;
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) {
      const float weight = fast_exp2(lse[n] - ref);
      sum += weight;
      o += part[n] * weight;
    }
  }
  const uint32_t hg = row / p.nodes, node = row - hg * p.nodes, hq = hkv * p.group + hg;
  if (column < p.d) store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + column, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
  if (column == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = top == -INFINITY && sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
}

// The runs' results of a row put together where there are many of them: a workgroup a row, whose threads have four columns of every
// RUNS-th run each, the first of them on their way while the runs' weights are found.  (attend_tree_join, a wavefront a row: 4 heads of
// 128 runs, 8 rows, 81 us; this 7.1, with those loads after the weights 7.6.)
template <typename T, int DPAD>
__device__ __forceinline__ void quantised_join_body(const TreeParams& p) {
  constexpr uint32_t COLUMNS = DPAD / 4, RUNS = 256 / COLUMNS;
  __shared__ float weights[256];
  __shared__ float of_wave[4];
  __shared__ f32x4 sums[RUNS][COLUMNS];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, head = blockIdx.x / p.rows, row = blockIdx.x - head * p.rows;
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv, column = tid % COLUMNS, of_runs = tid / COLUMNS;
  const TreeJoin join(p, head);
  if (join.count < 2) return;
  auto lse_of = [&](uint32_t s) { return s < join.count ? p.partial_lse[join.at(s, row)] : -INFINITY; };
  auto result_of = [&](uint32_t s) {
    return s < join.count && 4 * column < p.d ? *reinterpret_cast<const f32x4*>(p.partial_o + join.at(s, row) * p.d + 4 * column) : f32x4{0, 0, 0, 0};
  };
  float top = -INFINITY, sum = 0.0f;
  f32x4 o = {0, 0, 0, 0};
  auto add = [&](auto ahead) {
    constexpr uint32_t AHEAD = decltype(ahead)::value;
    const float first = lse_of(tid);
    f32x4 part[AHEAD];
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) part[n] = result_of(of_runs + RUNS * n);
    top = first;
    for (uint32_t s = 256 + tid; s < join.count; s += 256) top = fmaxf(top, lse_of(s));
    top = wave_max(top);
    if (lane == 0) of_wave[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
    // (a score that is no number makes its row one: the maximum passes it over)
    const float ref = top == -INFINITY ? 0.0f : top;
    for (uint32_t s0 = 0; s0 < join.count; s0 += 256) {
      __syncthreads();
      const float mine = s0 + tid < join.count ? fast_exp2((s0 == 0 ? first : lse_of(s0 + tid)) - ref) : 0.0f;
      weights[tid] = mine;
      sum += mine;
      __syncthreads();
      const uint32_t here = min(join.count - s0, 256u);
      for (uint32_t s = of_runs, n0 = 0; s < here; s += RUNS * AHEAD, n0 += AHEAD) {
        if (s0 + n0 > 0) {
#pragma unroll
          for (uint32_t n = 0; n < AHEAD; ++n) part[n] = result_of(s0 + s + RUNS * n);
        }
#pragma unroll
        for (uint32_t n = 0; n < AHEAD; ++n)
          if (s + RUNS * n < here) o += part[n] * weights[s + RUNS * n];
      }
    }
  };
  if (join.count <= 2 * RUNS) add(std::integral_constant<uint32_t, 2>{});
  else add(std::integral_constant<uint32_t, 8>{});
  sum = wave_sum(sum);
  __syncthreads();
  if (lane == 0) of_wave[wave] = sum;
  sums[of_runs][column] = o;
  __syncthreads();
  sum = of_wave[0] + of_wave[1] + of_wave[2] + of_wave[3];
  if (tid >= COLUMNS) return;
#pragma unroll
  for (uint32_t n = 1; n < RUNS; ++n) o += sums[n][column];
  const uint32_t hg = row / p.nodes, node = row - hg * p.nodes, hq = hkv * p.group + hg;
  if (4 * column < p.d) store4((T*)p.o.data + batch * p.o.sb + hq * p.o.sh + node * p.o.sn + 4 * column, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
  if (tid == 0 && p.lse) p.lse[((size_t)batch * p.hq + hq) * p.nodes + node] = top == -INFINITY && sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
}

}  // namespace attend
