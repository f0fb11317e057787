// Eight neighbouring bf16 channels of a row per lane, whatever the row's alignment and width.  A row of odd width starts
// anywhere in a 16-byte word; reading it two bytes at a time ran at a quarter of the memory bandwidth.  A lane instead reads
// the two aligned words that hold its eight channels (its neighbour reads the second one too: the L1 serves it) and
// shifts.  Such a word may reach over the row's ends into the pitch or the next row, where it is read and ignored; in the
// first and last rows it could reach over the ends of the operand, and they are read channel by channel.  The loads
// depend on nothing but addresses, so that a kernel can issue all of a row's before the first shift waits for one.
// Stores shift the other way, the missing channels coming from the lane before, and touch nothing outside the row.
// ALIGNED: rows start at 16-byte words and hold whole words (width a multiple of 8); then all of this is one access.
// (These rows are bound by instructions: what is done once a row has a branch of its own, what is done once a word has none.)
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace lc0b200 {

// Channels `by` .. `by` + 7 (0 <= by < 8) of the sixteen in a | b.
__device__ __forceinline__ uint4 shift_channels(const uint4& a, const uint4& b, int by) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t t[6], u[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) t[i] = (by & 4) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) u[i] = (by & 2) ? t[i + 1] : t[i];
  const int bits = (by & 1) * 16;
  return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits),
                    __funnelshift_r(u[3], u[4], bits));
}

// Channels between a 16-byte boundary and a row's start.
__device__ __forceinline__ int row_offset(const bf16* row) { return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) >> 1); }

struct RowWords {
  uint4 a, b;
};

// The word at row + at, put together from the row's own channels.
static __device__ __noinline__ uint4 edge_word(const bf16* row, int at, int width) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (at + j >= 0 && at + j < width) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[at + j]) << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Whether a word that holds a channel of this row lies within the operand, wherever it starts: seven channels may stick out.
__device__ __forceinline__ bool inner_row(long long row, long long rows, long long ld) {
  return row * ld >= 7 && (rows - 1 - row) * ld >= 7;
}

// The words of channels col .. col + 7 (col a multiple of 8); `inner` from inner_row.  Plain loads: a result may lie over its operand.
template <bool ALIGNED>
__device__ __forceinline__ RowWords load_words(const bf16* row, int col, int width, bool inner) {
  RowWords r;
  r.a = r.b = make_uint4(0u, 0u, 0u, 0u);
  const int at = ALIGNED ? col : col - row_offset(row);
  if (ALIGNED || inner) {
    if (col < width) r.a = *reinterpret_cast<const uint4*>(row + at);
    if (!ALIGNED && at + 8 < width) r.b = *reinterpret_cast<const uint4*>(row + at + 8);
  } else {
    if (col < width) r.a = edge_word(row, at, width);
    if (at + 8 < width) r.b = edge_word(row, at + 8, width);
  }
  return r;
}

// ... and the channels themselves, zeros past the row's end.
template <bool ALIGNED>
__device__ __forceinline__ uint4 channels_of(const RowWords& r, const bf16* row, int col, int width) {
  if (ALIGNED) return r.a;
  uint4 v = shift_channels(r.a, r.b, row_offset(row));
  const int valid = width - col;
  if (valid < 8) {
    v.x &= valid >= 2 ? 0xFFFFFFFFu : (valid == 1 ? 0xFFFFu : 0u);
    v.y &= valid >= 4 ? 0xFFFFFFFFu : (valid == 3 ? 0xFFFFu : 0u);
    v.z &= valid >= 6 ? 0xFFFFFFFFu : (valid == 5 ? 0xFFFFu : 0u);
    v.w &= valid == 7 ? 0xFFFFu : 0u;
  }
  return v;
}

__device__ __forceinline__ void store_channels(bf16* row, int col, const uint4& v, int first, int end) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= first && j < end) reinterpret_cast<uint16_t*>(row)[col + j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
  }
}

// Stores this lane's channels col .. col + 7 (lane i's col is lane 0's plus 8 i) as far as they lie inside the row.  Every
// lane of the warp takes part.  A warp walks a run of the row, 256 channels a step: `carry` takes the last lane's channels
// from one step to the next, `begin` and `end` mark the run's first and last step.
template <bool ALIGNED>
__device__ __forceinline__ void store8_row(bf16* row, int col, int width, const uint4& v, uint4& carry, bool begin, bool end) {
  const int valid = width - col;
  if (ALIGNED) {
    if (valid > 0) *reinterpret_cast<uint4*>(row + col) = v;
    return;
  }
  const int off = row_offset(row);
  if (off == 0) {  // the same for the warp
    if (valid >= 8) *reinterpret_cast<uint4*>(row + col) = v;
    else store_channels(row, col, v, 0, valid);
    return;
  }
  const int lane = threadIdx.x & 31;
  uint4 before;
  before.x = __shfl_sync(0xFFFFFFFFu, v.x, (lane + 31) & 31);
  before.y = __shfl_sync(0xFFFFFFFFu, v.y, (lane + 31) & 31);
  before.z = __shfl_sync(0xFFFFFFFFu, v.z, (lane + 31) & 31);
  before.w = __shfl_sync(0xFFFFFFFFu, v.w, (lane + 31) & 31);
  const uint4 last = before;
  if (lane == 0) before = carry;
  carry = last;
  if (valid <= 0) return;
  // The aligned word that ends inside this lane's channels: the last `off` of the lane before, then its own.
  const uint4 word = shift_channels(before, v, 8 - off);
  const bool first = begin && lane == 0;
  if (!first && valid + off >= 8) *reinterpret_cast<uint4*>(row + col - off) = word;
  else store_channels(row, col - off, word, first ? off : 0, valid + off);
  // The last `off` channels are the next lane's to store, where there is one.
  if (valid <= 8 || (end && lane == 31)) store_channels(row, col, v, 8 - off, valid);
}

}  // namespace lc0b200
