// Entries of least accumulated weight leave a cache.  evict_select: which slots of a (sequence, key head) stay, in order; a
// workgroup each.  evict_gather: their rows of K and V move to the new cache, 16 bytes a lane.  evict_whole: both.
//
// Selection by radix: the weights as unsigned integers of the same order, three passes over 11, 11 and 10 bits, each a
// histogram of the candidates that agree with the digits found so far.  What is left is the exact weight of the last entry that
// stays and how many of that weight do; ties go to the lowest slots.  A second walk writes the slots in order, every wavefront a
// run of its own whose place is known from the counts before it.
//
// Measured, 16 x 8 heads of up to 8192 entries cut to 2048, 128 bf16 columns (266 MB): selection 13 us, bound by its chain of passes and
// barriers (read anew in every pass, digits looked through by one wavefront: 23); gather 43 us, bound by memory, 6 TB/s.
#pragma once
#include "attend_tree.h"

namespace attend {

// a weight as an integer that orders as the weight does; no number comes last
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t bits = __builtin_bit_cast(uint32_t, w + 0.0f);  // (-0 is 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ void evict_select_body(const EvictParams& p) {
  constexpr uint32_t THREADS = 1024, WAVES = THREADS / 64, KEPT = 16;
  __shared__ uint32_t bins[2048];
  __shared__ uint32_t shared_prefix, shared_left;
  __shared__ uint32_t shared_more[WAVES], shared_same[WAVES];
  const uint32_t head = blockIdx.x, batch = head / p.hkv, tid = threadIdx.x, lane = tid & 63, wave = tid / 64;
  const int given = p.lengths[batch];
  const uint32_t n = given < 0 ? 0 : min((uint32_t)given, p.max_length);
  const uint32_t held = min(n, p.keep);
  if (tid == 0 && head == batch * p.hkv) p.lengths_out[batch] = (int)held;
  const float* weights = p.weights + (int64_t)head * p.weights_stride;
  const int* positions = p.positions ? p.positions + (int64_t)head * p.positions_stride : nullptr;
  float* weights_out = p.weights_out + (int64_t)head * p.out_stride;
  int* positions_out = p.positions_out + (int64_t)head * p.out_stride;
  int* chosen = p.chosen + (int64_t)head * p.keep;
  auto stay = [&](uint32_t to, uint32_t slot, float weight) {
    chosen[to] = (int)slot;
    weights_out[to] = weight;
    positions_out[to] = positions ? positions[slot] : (int)slot;
  };
  // the last `recent` stay whatever their weight (all of them where nothing has to go)
  const uint32_t recent = n <= p.keep ? held : p.recent, old = n - recent, want = held - recent;
  for (uint32_t i = tid; i < recent; i += THREADS) stay(want + i, old + i, weights[old + i]);
  if (want == 0) return;

  // a wavefront's run of the weights, 64 at a time: the first ones stay in registers for all passes
  const uint32_t rounds = (old + THREADS - 1) / THREADS, begin = min(wave * rounds * 64, old), end = min(begin + rounds * 64, old);
  float kept[KEPT];
#pragma unroll
  for (uint32_t j = 0; j < KEPT; ++j) kept[j] = begin + 64 * j + lane < end ? weights[begin + 64 * j + lane] : 0.0f;
  auto each_kept = [&](auto use) {
#pragma unroll
    for (uint32_t j = 0; j < KEPT; ++j)
      if (j < rounds) use(begin + 64 * j + lane, kept[j]);
  };
  auto each = [&](auto use) {
    each_kept(use);
#pragma unroll 4
    for (uint32_t j = KEPT; j < rounds; ++j) {
      const uint32_t i = begin + 64 * j + lane;
      use(i, i < end ? weights[i] : 0.0f);
    }
  };

  uint32_t prefix = 0, mask = 0, left = want;  // digits found, the bits they cover, how many of them are still wanted
  for (int pass = 0; pass < 3; ++pass) {
    const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 1024 : 2048;
    bins[tid] = bins[tid + THREADS] = 0;
    __syncthreads();
    each([&](uint32_t i, float weight) {
      const uint32_t key = weight_key(weight);
      if (i < end && (key & mask) == prefix) atomicAdd(&bins[key >> shift & (width - 1)], 1u);
    });
    __syncthreads();
    // a thread's two digits, the largest first; how many candidates have larger ones
    const uint32_t top = 2047 - 2 * tid, first = bins[top], second = bins[top - 1];
    uint32_t upto = first + second;
#pragma unroll
    for (int bit = 1; bit < 64; bit <<= 1) {
      const uint32_t other = __shfl_up(upto, bit);
      if ((int)lane >= bit) upto += other;
    }
    if (lane == 63) shared_more[wave] = upto;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) upto += w < wave ? shared_more[w] : 0;
    const uint32_t above = upto - first - second;
    if (above < left && upto >= left) {
      const bool in_first = above + first >= left;
      shared_prefix = prefix | (in_first ? top : top - 1) << shift;
      shared_left = left - above - (in_first ? 0 : first);
    }
    __syncthreads();
    prefix = shared_prefix;
    left = shared_left;
    mask |= (width - 1) << shift;
  }

  uint32_t more = 0, same = 0;
  each([&](uint32_t i, float weight) {
    const uint32_t key = weight_key(weight);
    more += i < end && key > prefix;
    same += i < end && key == prefix;
  });
#pragma unroll
  for (int bit = 1; bit < 64; bit <<= 1) {
    more += __shfl_xor(more, bit);
    same += __shfl_xor(same, bit);
  }
  __syncthreads();
  if (lane == 0) {
    shared_more[wave] = more;
    shared_same[wave] = same;
  }
  __syncthreads();
  uint32_t more_before = 0, same_before = 0;
  for (uint32_t w = 0; w < wave; ++w) {
    more_before += shared_more[w];
    same_before += shared_same[w];
  }
  uint32_t to = more_before + min(same_before, left);
  const uint64_t below = (1ull << lane) - 1;
  auto place = [&](uint32_t i, float weight) {
    const uint32_t key = weight_key(weight);
    const bool is_same = i < end && key == prefix;
    const uint64_t sames = __builtin_amdgcn_ballot_w64(is_same);
    const bool stays = i < end && (key > prefix || (is_same && same_before + __popcll(sames & below) < left));
    const uint64_t stayers = __builtin_amdgcn_ballot_w64(stays);
    if (stays) stay(to + __popcll(stayers & below), i, weight);
    to += __popcll(stayers);
    same_before += __popcll(sames);
  };
  each_kept(place);
  for (uint32_t j = KEPT; j < rounds; ++j) {  // (one after the other: a round's places follow from the one before)
    const uint32_t i = begin + 64 * j + lane;
    place(i, i < end ? weights[i] : 0.0f);
  }
}

// 64 rows that stay, K and V, by THREADS threads (a row whose new page the cache does not have goes nowhere)
template <uint32_t THREADS>
__device__ __forceinline__ void evict_move(const EvictParams& p, uint32_t element, uint32_t head, uint32_t row0, int64_t (*offsets)[4], bool* goes) {
  const uint32_t batch = head / p.hkv, hkv = head - batch * p.hkv, tid = threadIdx.x;
  const int given = p.lengths[batch];
  const uint32_t n = given < 0 ? 0 : min((uint32_t)given, p.max_length), held = min(n, p.keep);
  if (row0 >= held) return;
  const uint32_t count = min(held - row0, 64u);
  if (tid < count) {
    const uint32_t from = (uint32_t)p.chosen[(int64_t)head * p.keep + row0 + tid], to = row0 + tid;
    const uint32_t from_index = from / p.from.page, from_slot = from - from_index * p.from.page;
    const uint32_t to_index = to / p.to.page, to_slot = to - to_index * p.to.page;
    const int64_t from_page = page_of(p.from, batch, from_index), to_page = page_if_any(p.to, batch, to_index);
    goes[tid] = to_page >= 0;
    offsets[tid][0] = (from_page * p.from.k_page + hkv * p.from.k_head + from_slot * p.from.k_slot) * element;
    offsets[tid][1] = (to_page * p.to.k_page + hkv * p.to.k_head + to_slot * p.to.k_slot) * element;
    offsets[tid][2] = (from_page * p.from.v_page + hkv * p.from.v_head + from_slot * p.from.v_slot) * element;
    offsets[tid][3] = (to_page * p.to.v_page + hkv * p.to.v_head + to_slot * p.to.v_slot) * element;
  }
  __syncthreads();
  const uint32_t per_row = p.row_bytes / 16, items = count * per_row;
#pragma unroll 4
  for (uint32_t i = tid; i < items; i += THREADS) {
    const uint32_t row = i / per_row, c = 16 * (i - row * per_row);
    if (!goes[row]) continue;
    const u32x4 k = ldg128((const char*)p.from.k + offsets[row][0] + c), v = ldg128((const char*)p.from.v + offsets[row][2] + c);
    *reinterpret_cast<u32x4*>((char*)p.to.k + offsets[row][1] + c) = k;
    *reinterpret_cast<u32x4*>((char*)p.to.v + offsets[row][3] + c) = v;
  }
}

__device__ __forceinline__ void evict_gather_body(const EvictParams& p, uint32_t element) {
  __shared__ int64_t offsets[64][4];  // K from, K to, V from, V to; bytes
  __shared__ bool goes[64];
  const uint32_t head = blockIdx.x / p.tiles;
  evict_move<256>(p, element, head, (blockIdx.x - head * p.tiles) * 64, offsets, goes);
}

// both in one launch, for caches that are small after it
__device__ __forceinline__ void evict_whole_body(const EvictParams& p, uint32_t element) {
  __shared__ int64_t offsets[64][4];
  __shared__ bool goes[64];
  evict_select_body(p);
  for (uint32_t tile = 0; tile < p.tiles; ++tile) {
    __syncthreads();  // (the slots are written, the offsets before are read)
    evict_move<1024>(p, element, blockIdx.x, tile * 64, offsets, goes);
  }
}

}  // namespace attend
