// Rows of bf16 that start at any two-byte boundary and have any width.  A warp walks a run of the row 64 channels a step;
// in step s lane l holds the pair of channels c = run + 64 s + 2 l and c + 1.  Memory is touched in aligned four-byte words:
// where the row starts in the middle of one, a lane's pair is the upper half of its own word and the lower half of the
// next lane's, one shuffle and one funnel shift.  (Single channels ran at a quarter of the memory bandwidth; shifting
// eight channels between 16-byte words took three times as many instructions as this and was bound by them.)
// A word may hold one channel's room before the row or behind it, which is read and ignored; the rows where that could lie
// outside the operand are read channel by channel.  Nothing outside the row is written.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace lc0b200 {

// 1 where the row starts in the upper half of a four-byte word.
__device__ __forceinline__ int row_half(const bf16* row) { return static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 1) & 1u); }

// Whether one channel's room on either side of the row lies within the operand.
__device__ __forceinline__ bool inner_row(long long row, long long rows, long long ld) { return row > 0 && row + 1 < rows && ld > 0; }

// The word of channels c - half, c - half + 1, whose own room is 0 <= channel < width.
__device__ __forceinline__ uint32_t load_row_word(const bf16* row, int c, int half, int width, bool inner) {
  if (c - half >= width) return 0u;
  if (inner) return *reinterpret_cast<const uint32_t*>(row + c - half);
  const uint16_t* channels = reinterpret_cast<const uint16_t*>(row);
  const uint32_t lo = c - half >= 0 ? channels[c - half] : 0u;
  const uint32_t hi = c - half + 1 < width ? channels[c - half + 1] : 0u;
  return lo | (hi << 16);
}

// STEPS steps of words from channel `run` on, and the word behind them (lane 0's); plain loads: a result may lie over its operand.
template <int STEPS>
__device__ __forceinline__ void load_row_words(uint32_t (&w)[STEPS + 1], const bf16* row, int run, int width, bool inner) {
  const int lane = threadIdx.x & 31, half = row_half(row);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) w[s] = load_row_word(row, run + 64 * s + 2 * lane, half, width, inner);
  w[STEPS] = lane == 0 && half != 0 ? load_row_word(row, run + 64 * STEPS, half, width, inner) : 0u;
}

// The pair of step s; channels past the row's end hold anything.  Every lane takes part.
template <int STEPS>
__device__ __forceinline__ uint32_t row_pair(const uint32_t (&w)[STEPS + 1], int s, int half) {
  const int lane = threadIdx.x & 31;
  // Lane 31's next word is lane 0's of the next step: the source lane sends the one that its reader needs.
  const uint32_t next = __shfl_sync(0xFFFFFFFFu, lane == 0 ? w[s + 1] : w[s], (lane + 1) & 31);
  return __funnelshift_r(w[s], next, 16 * half);
}

// Stores the pair of channels c, c + 1 as far as they lie in the row.  `carry` takes lane 31's pair to the next step; `begin`,
// `end`: the first and last step of this warp's run.  Every lane takes part.
__device__ __forceinline__ void store_row_pair(bf16* row, int c, int half, int width, uint32_t pair, uint32_t& carry, bool begin, bool end) {
  uint16_t* channels = reinterpret_cast<uint16_t*>(row);
  if (half == 0) {  // the same for the warp
    if (c + 1 < width) *reinterpret_cast<uint32_t*>(row + c) = pair;
    else if (c < width) channels[c] = static_cast<uint16_t>(pair);
    return;
  }
  const int lane = threadIdx.x & 31;
  const uint32_t turned = __shfl_sync(0xFFFFFFFFu, pair, (lane + 31) & 31);
  const uint32_t before = lane == 0 ? carry : turned;
  carry = turned;  // lane 0 now holds this step's lane 31
  const bool first = begin && lane == 0;
  if (c < width && !first) *reinterpret_cast<uint32_t*>(row + c - 1) = __funnelshift_r(before, pair, 16);
  else if (first && c < width) channels[c] = static_cast<uint16_t>(pair);
  // A channel c + 1 that no other lane's word holds: the row's last, or the run's.
  if ((c + 2 == width || (end && lane == 31)) && c + 1 < width) channels[c + 1] = static_cast<uint16_t>(pair >> 16);
}

}  // namespace lc0b200
