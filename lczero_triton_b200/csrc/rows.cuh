// Eight neighbouring bf16 channels of a row per lane, whatever the row's alignment and width.  A row of odd width starts
// anywhere in a 16-byte word; reading it two bytes at a time ran at a quarter of the memory bandwidth.  A lane instead reads
// the two aligned words that hold its eight channels (its neighbour reads the second one too: the L1 serves it) and
// shifts.  Such a word may reach over the row's ends into the pitch or the next row, where it is read and ignored, but
// never over the ends of the whole operand: there it is put together channel by channel.  The loads depend on nothing
// but addresses, so that a kernel can issue all of a row's before the first shift waits for one.
// Stores shift the other way, the missing channels coming from the lane before, and touch nothing outside the row.
// ALIGNED: rows start at 16-byte words and hold whole words (width a multiple of 8); then all of this is one access.
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

// One aligned word at row + at, of which the channels 0 <= at + j < width belong to the row; [first, end) is the operand.
__device__ __forceinline__ uint4 load_word(const bf16* row, int at, int width, const bf16* first, const bf16* end) {
  const bf16* word = row + at;
  if (word >= first && word + 8 <= end) return *reinterpret_cast<const uint4*>(word);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (at + j >= 0 && at + j < width) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[at + j]) << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The words of channels col .. col + 7 (col a multiple of 8).  Plain loads: a result may lie over its operand.
template <bool ALIGNED>
__device__ __forceinline__ RowWords load_words(const bf16* row, int col, int width, const bf16* first, const bf16* end) {
  RowWords r;
  r.a = r.b = make_uint4(0u, 0u, 0u, 0u);
  if (ALIGNED) {
    if (col < width) r.a = *reinterpret_cast<const uint4*>(row + col);
    return r;
  }
  const int at = col - row_offset(row);
  if (col < width) r.a = load_word(row, at, width, first, end);
  if (at != col && at + 8 < width) r.b = load_word(row, at + 8, width, first, end);
  return r;
}

// ... and the channels themselves, zeros past the row's end.
template <bool ALIGNED>
__device__ __forceinline__ uint4 channels_of(const RowWords& r, const bf16* row, int col, int width) {
  if (ALIGNED) return r.a;
  const uint4 v = shift_channels(r.a, r.b, row_offset(row));
  const int valid = width - col;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] &= valid >= 2 * i + 2 ? 0xFFFFFFFFu : (valid == 2 * i + 1 ? 0xFFFFu : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void store_channels(bf16* row, int col, const uint4& v, int first, int end) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= first && j < end) reinterpret_cast<uint16_t*>(row)[col + j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
  }
}

// Stores this lane's channels col .. col + 7 (lane i's col is lane 0's plus 8 i) as far as they lie inside the row.  Every
// lane of the warp takes part.
template <bool ALIGNED>
__device__ __forceinline__ void store8_row(bf16* row, int col, int width, const uint4& v) {
  const int off = ALIGNED ? 0 : row_offset(row);
  const int valid = width - col;
  if (off == 0) {  // the same for the warp
    if (valid >= 8) *reinterpret_cast<uint4*>(row + col) = v;
    else if (!ALIGNED) store_channels(row, col, v, 0, valid);
    return;
  }
  const int lane = threadIdx.x & 31;
  uint4 before;
  before.x = __shfl_up_sync(0xFFFFFFFFu, v.x, 1);
  before.y = __shfl_up_sync(0xFFFFFFFFu, v.y, 1);
  before.z = __shfl_up_sync(0xFFFFFFFFu, v.z, 1);
  before.w = __shfl_up_sync(0xFFFFFFFFu, v.w, 1);
  if (valid <= 0) return;
  // The aligned word that ends inside this lane's channels: the last `off` of the lane before, then its own.
  const uint4 word = shift_channels(before, v, 8 - off);
  const int word_valid = valid + off;
  if (lane > 0 && word_valid >= 8) *reinterpret_cast<uint4*>(row + col - off) = word;
  else store_channels(row, col - off, word, lane > 0 ? 0 : off, word_valid);
  // The last `off` channels are the next lane's to store, where there is one.
  if (lane == 31 || valid <= 8) store_channels(row, col, v, 8 - off, valid);
}

}  // namespace lc0b200
