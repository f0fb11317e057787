// bf16 to e4m3 with one f32 scale per block (the rule is in fp8.cuh): 1 x 128 blocks along a row for activations,
// 128 x 128 tiles for weights.  HBM-bound: three bytes an element move (two in, one out) and the values stay in
// registers between the maximum and the rounding.
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace lc0b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 16;  // a half-warp (16 lanes x 8 values) holds one 1 x 128 block

// Magnitudes of bf16 values order as 16-bit unsigned integers (NaN above infinity): packed maximum of eight.
__device__ __forceinline__ uint32_t packed_magnitude(const uint4& raw) {
  return __vmaxu2(__vmaxu2(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu), __vmaxu2(raw.z & 0x7FFF7FFFu, raw.w & 0x7FFF7FFFu));
}
// The larger half of a packed maximum as float bits.
__device__ __forceinline__ uint32_t magnitude_of_packed(uint32_t m) { return max(m & 0xFFFFu, m >> 16) << 16; }

template <bool WORDS>
__device__ __forceinline__ void store_codes(uint8_t* row, int col, int width, const uint4& raw, float inverse) {
  const float2 a = unpack_bf16x2(raw.x), b = unpack_bf16x2(raw.y), c = unpack_bf16x2(raw.z), d = unpack_bf16x2(raw.w);
  const uint32_t lo = fp8_pack4(a.x * inverse, a.y * inverse, b.x * inverse, b.y * inverse);
  const uint32_t hi = fp8_pack4(c.x * inverse, c.y * inverse, d.x * inverse, d.y * inverse);
  const int valid = width - col;
  if (WORDS && valid >= 8) {
    *reinterpret_cast<uint2*>(row + col) = make_uint2(lo, hi);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < valid) row[col + j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

// A half-warp takes UNROLL neighbouring blocks of one row; a CTA 16 rows.
template <int UNROLL, bool ALIGNED, bool WORDS>
__global__ void __launch_bounds__(kThreads)
quantize_fp8_rows_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                         int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane16 = threadIdx.x & 15;
  const long long row = blockIdx.x * static_cast<long long>(kRowsPerCta) + (threadIdx.x >> 4);
  const bool row_ok = row < rows;  // the other half of the warp may have a row: nobody leaves before the shuffles
  const bf16* src = x + row * ld_in;
  uint8_t* dst = q_out + row * ld_out;
  const int blocks = static_cast<int>(ceil_div_ll(width, kFp8Block));
  for (int first = blockIdx.y * UNROLL; first < blocks; first += gridDim.y * UNROLL) {
    RowWords words[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      words[u].a = words[u].b = make_uint4(0u, 0u, 0u, 0u);
      if (row_ok && first + u < blocks) words[u] = load_words<ALIGNED>(src, (first + u) * kFp8Block + lane16 * 8, width, inner_row(row, rows, ld_in));
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const uint4 raw = channels_of<ALIGNED>(words[u], src, (first + u) * kFp8Block + lane16 * 8, width);
      uint32_t m = packed_magnitude(raw);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      float scale, inverse;
      fp8_block_scale(magnitude_of_packed(m), scale, inverse);
      const int block = first + u;
      if (row_ok && block < blocks) {
        if (lane16 == 0) scale_out[block * ld_scale + row] = scale;
        store_codes<WORDS>(dst, block * kFp8Block + lane16 * 8, width, raw, inverse);
      }
    }
  }
}

// One CTA per 128 x 128 tile: each half-warp holds eight rows of the tile.
template <bool ALIGNED, bool WORDS>
__global__ void __launch_bounds__(kThreads)
quantize_fp8_tiles_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                          int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ uint32_t warp_max[2][kThreads / 32];
  constexpr int kRowsPerThread = kFp8Block / kRowsPerCta;
  const int lane16 = threadIdx.x & 15, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * kFp8Block + lane16 * 8;
  const long long row_tiles = ceil_div_ll(rows, kFp8Block);
  int parity = 0;
  for (long long tile = blockIdx.y; tile < row_tiles; tile += gridDim.y, parity ^= 1) {
    const long long row0 = tile * kFp8Block + (threadIdx.x >> 4);
    RowWords words[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const long long row = row0 + i * kRowsPerCta;
      words[i].a = words[i].b = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows) words[i] = load_words<ALIGNED>(x + row * ld_in, col, width, inner_row(row, rows, ld_in));
    }
    uint4 raw[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) raw[i] = channels_of<ALIGNED>(words[i], x + (row0 + i * kRowsPerCta) * ld_in, col, width);
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) m = __vmaxu2(m, packed_magnitude(raw[i]));
    m = __reduce_max_sync(0xFFFFFFFFu, magnitude_of_packed(m));
    if ((threadIdx.x & 31) == 0) warp_max[parity][warp] = m;
    __syncthreads();  // two sets of words in turn: the next tile's writes cannot overtake this tile's reads
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, warp_max[parity][w]);
    float scale, inverse;
    fp8_block_scale(m, scale, inverse);
    if (threadIdx.x == 0) scale_out[tile * ld_scale + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const long long row = row0 + i * kRowsPerCta;
      if (row < rows) store_codes<WORDS>(q_out + row * ld_out, col, width, raw[i], inverse);
    }
  }
}

}  // namespace

int quantize_fp8(void* out, float* scale, const void* in, long long rows, int width, int block_rows, long long ld_in,
                 long long ld_out, long long ld_scale, cudaStream_t st) {
  auto* q = reinterpret_cast<uint8_t*>(out);
  const auto* x = reinterpret_cast<const bf16*>(in);
  const bool aligned = aligned16(in) && (ld_in % 8) == 0 && (width % 8) == 0;
  const bool words = (reinterpret_cast<uintptr_t>(out) % 8) == 0 && (ld_out % 8) == 0;
  const long long blocks = ceil_div_ll(width, kFp8Block);
  const dim3 threads(kThreads);
  if (block_rows == 1) {
    constexpr int kUnroll = 4;
    const long long groups = ceil_div_ll(blocks, kUnroll);
    const dim3 grid(static_cast<unsigned>(ceil_div_ll(rows, kRowsPerCta)), static_cast<unsigned>(groups < 65535 ? groups : 65535));
    if (aligned && words) launch_dependent(quantize_fp8_rows_kernel<kUnroll, true, true>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    else if (words) launch_dependent(quantize_fp8_rows_kernel<kUnroll, false, true>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    else launch_dependent(quantize_fp8_rows_kernel<kUnroll, false, false>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    return launch_status();
  }
  const long long row_tiles = ceil_div_ll(rows, kFp8Block);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(row_tiles < 65535 ? row_tiles : 65535));
  if (aligned && words) launch_dependent(quantize_fp8_tiles_kernel<true, true>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  else if (words) launch_dependent(quantize_fp8_tiles_kernel<false, true>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  else launch_dependent(quantize_fp8_tiles_kernel<false, false>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  return launch_status();
}

}  // namespace lc0b200
