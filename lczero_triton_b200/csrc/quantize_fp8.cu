// bf16 to e4m3 with one f32 scale per block (the rule is in fp8.cuh): 1 x 128 blocks along a row for activations,
// 128 x 128 tiles for weights.  HBM-bound: three bytes an element move (two in, one out) and the values stay in
// registers between the maximum and the rounding.  Aligned: 262144 x 1536 in 182 us (6.7 TB/s), 8190 x 8200 as tiles in 37
// (5.4); any alignment: 65536 x 1001 in 52 us (3.8 TB/s).
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace lc0b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 16;  // a half-warp (16 lanes x 8 values) holds one 1 x 128 block

// Rows of whole, aligned 16-byte words: a half-warp takes four neighbouring blocks of one row, a CTA 16 rows.  (With every
// lane reducing and dividing for all four blocks the kernel was bound by its instructions: 262144 x 1536 in 203 us.)
__global__ void __launch_bounds__(kThreads)
quantize_fp8_rows_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                         int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane16 = threadIdx.x & 15, mine = lane16 >> 2;
  const long long row = blockIdx.x * static_cast<long long>(kRowsPerCta) + (threadIdx.x >> 4);
  const int groups = row < rows ? width >> 3 : 0;  // a half-warp without a row stays for the other half's shuffles
  const uint4* src = reinterpret_cast<const uint4*>(x + row * ld_in);
  uint2* dst = reinterpret_cast<uint2*>(q_out + row * ld_out);
  const int blocks = static_cast<int>(ceil_div_ll(width, kFp8Block));
  for (int first = blockIdx.y * 4; first < blocks; first += gridDim.y * 4) {
    uint4 raw[4];
    uint32_t m[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int idx = (first + u) * 16 + lane16;
      raw[u] = idx < groups ? __ldg(src + idx) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) m[u] = magnitude_of_packed(packed_magnitude(raw[u]));
    float scale, inverse;
    fp8_block_scale(max_of_four_blocks(m), scale, inverse);
    if ((lane16 & 3) == 0 && row < rows && first + mine < blocks) scale_out[(first + mine) * ld_scale + row] = scale;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int idx = (first + u) * 16 + lane16;
      const float factor = from_block(inverse, u);
      if (idx < groups) dst[idx] = codes8(raw[u], factor);
    }
  }
}

// Rows of any alignment and width: a warp takes UNROLL neighbouring blocks of a row, channel lane + 32 i of a block to a lane.
// FULL: all of them lie inside the row, nothing is checked per channel.
template <int UNROLL, bool FULL>
__device__ __forceinline__ void quantize_run(uint8_t* dst, float* scales, long long ld_scale, const bf16* src, int run, int width) {
  const int lane = threadIdx.x & 31;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(src) + run + lane;
  uint8_t* q = dst + run + lane;
  uint32_t raw[UNROLL][4];  // bf16 bits
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = kFp8Block * u + 32 * i;
      raw[u][i] = FULL || run + at + lane < width ? __ldg(x + at) : 0u;
    }
  }
  // Lane u works out block u's scale (two divisions once, not UNROLL times).
  uint32_t mine = 0u;
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const uint32_t m = max(max(raw[u][0] & 0x7FFFu, raw[u][1] & 0x7FFFu), max(raw[u][2] & 0x7FFFu, raw[u][3] & 0x7FFFu));
    const uint32_t block = __reduce_max_sync(0xFFFFFFFFu, m);
    mine = lane == u ? block : mine;
  }
  float scale, inverse;
  fp8_block_scale(mine << 16, scale, inverse);
  if (lane < UNROLL && (FULL || run + kFp8Block * lane < width)) scales[(run / kFp8Block + lane) * ld_scale] = scale;
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const float factor = __shfl_sync(0xFFFFFFFFu, inverse, u);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const int at = kFp8Block * u + 32 * i;
      const uint16_t codes = fp8_pack2(__uint_as_float(raw[u][i] << 16) * factor, __uint_as_float(raw[u][i + 1] << 16) * factor);
      if (FULL || run + at + lane < width) q[at] = static_cast<uint8_t>(codes);
      if (FULL || run + at + 32 + lane < width) q[at + 32] = static_cast<uint8_t>(codes >> 8);
    }
  }
}

template <int UNROLL>
__global__ void __launch_bounds__(kThreads)
quantize_fp8_odd_rows_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                             int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  const long long row = blockIdx.x * static_cast<long long>(kThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  constexpr int kRun = UNROLL * kFp8Block;
  for (int run = blockIdx.y * kRun; run < width; run += gridDim.y * kRun) {
    if (run + kRun <= width) quantize_run<UNROLL, true>(q_out + row * ld_out, scale_out + row, ld_scale, x + row * ld_in, run, width);
    else quantize_run<UNROLL, false>(q_out + row * ld_out, scale_out + row, ld_scale, x + row * ld_in, run, width);
  }
}

// The maximum over a CTA's threads of magnitude bits.  `words` (one per warp) is used for every other tile only, so that the
// next tile's writes cannot overtake this tile's reads.
__device__ __forceinline__ uint32_t cta_max(uint32_t m, uint32_t* words) {
  const int lane = threadIdx.x & 31;
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (lane == 0) words[threadIdx.x >> 5] = m;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < kThreads / 32 ? words[lane] : 0u);
}

// One CTA per 128 x 128 tile, whole aligned words: each half-warp holds eight rows of the tile.
__global__ void __launch_bounds__(kThreads)
quantize_fp8_tiles_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                          int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ uint32_t warp_max[2][kThreads / 32];
  constexpr int kRowsPerThread = kFp8Block / kRowsPerCta;
  const int col = blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
  const long long row_tiles = ceil_div_ll(rows, kFp8Block);
  int parity = 0;
  for (long long tile = blockIdx.y; tile < row_tiles; tile += gridDim.y, parity ^= 1) {
    const long long row0 = tile * kFp8Block + (threadIdx.x >> 4);
    uint4 raw[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const long long row = row0 + i * kRowsPerCta;
      raw[i] = row < rows && col < width ? __ldg(reinterpret_cast<const uint4*>(x + row * ld_in + col)) : make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) m = __vmaxu2(m, packed_magnitude(raw[i]));
    float scale, inverse;
    fp8_block_scale(cta_max(magnitude_of_packed(m), warp_max[parity]), scale, inverse);
    if (threadIdx.x == 0) scale_out[tile * ld_scale + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const long long row = row0 + i * kRowsPerCta;
      if (row < rows && col < width) *reinterpret_cast<uint2*>(q_out + row * ld_out + col) = codes8(raw[i], inverse);
    }
  }
}

// ... and for rows of any alignment and width: a warp holds every eighth row of the tile, channel lane + 32 i to a lane.
// Bound by the number of memory instructions (a channel each).  Four CTAs an SM, one's loads overlap another's stores:
// 174775 x 846 in 108 us, 592 with one (175 registers a thread), 125 with three of 512 threads.  FULL: the tile lies
// inside the matrix, nothing is checked per channel (215 us with the checks).
constexpr int kOddCtas = 4;

template <bool FULL>
__device__ __forceinline__ void quantize_odd_tile(uint8_t* q, float* scale_out, const uint16_t* x, uint32_t* words, long long rows,
                                                  int width, long long ld_in, long long ld_out) {
  constexpr int kWarps = kThreads / 32, kRowsPerWarp = kFp8Block / kWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint16_t* src = x + warp * ld_in + lane;
  uint32_t raw[kRowsPerWarp][2];  // bf16 bits, two channels to a word
  uint32_t m = 0u;
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r, src += kWarps * ld_in) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = FULL || (warp + kWarps * r < rows && lane + 32 * i < width) ? __ldg(src + 32 * i) : 0u;
    raw[r][0] = v[0] | (v[1] << 16);
    raw[r][1] = v[2] | (v[3] << 16);
  }
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) m = __vmaxu2(m, __vmaxu2(raw[r][0] & 0x7FFF7FFFu, raw[r][1] & 0x7FFF7FFFu));
  float scale, inverse;
  fp8_block_scale(cta_max(magnitude_of_packed(m), words), scale, inverse);
  if (threadIdx.x == 0) *scale_out = scale;
  uint8_t* dst = q + warp * ld_out + lane;
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r, dst += kWarps * ld_out) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 v = unpack_bf16x2(raw[r][i]);
      const uint16_t codes = fp8_pack2(v.x * inverse, v.y * inverse);
      if (FULL || (warp + kWarps * r < rows && lane + 64 * i < width)) dst[64 * i] = static_cast<uint8_t>(codes);
      if (FULL || (warp + kWarps * r < rows && lane + 64 * i + 32 < width)) dst[64 * i + 32] = static_cast<uint8_t>(codes >> 8);
    }
  }
}

__global__ void __launch_bounds__(kThreads, kOddCtas)
quantize_fp8_odd_tiles_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                              int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ uint32_t warp_max[2][kThreads / 32];
  const int c0 = blockIdx.x * kFp8Block;
  const long long row_tiles = ceil_div_ll(rows, kFp8Block);
  int parity = 0;
  for (long long tile = blockIdx.y; tile < row_tiles; tile += gridDim.y, parity ^= 1) {
    const long long row0 = tile * kFp8Block;
    uint8_t* q = q_out + row0 * ld_out + c0;
    float* scale = scale_out + tile * ld_scale + blockIdx.x;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(x) + row0 * ld_in + c0;
    if (row0 + kFp8Block <= rows && c0 + kFp8Block <= width) {
      quantize_odd_tile<true>(q, scale, src, warp_max[parity], kFp8Block, kFp8Block, ld_in, ld_out);
    } else {
      quantize_odd_tile<false>(q, scale, src, warp_max[parity], rows - row0, width - c0, ld_in, ld_out);
    }
  }
}

}  // namespace

int quantize_fp8(void* out, float* scale, const void* in, long long rows, int width, int block_rows, long long ld_in,
                 long long ld_out, long long ld_scale, cudaStream_t st) {
  auto* q = reinterpret_cast<uint8_t*>(out);
  const auto* x = reinterpret_cast<const bf16*>(in);
  const bool aligned = (width % 8) == 0 && aligned16(in) && (ld_in % 8) == 0 && (reinterpret_cast<uintptr_t>(out) % 8) == 0 && (ld_out % 8) == 0;
  const long long blocks = ceil_div_ll(width, kFp8Block);
  const dim3 threads(kThreads);
  auto capped = [](long long count) { return static_cast<unsigned>(count < 65535 ? count : 65535); };
  if (block_rows == 1) {
    constexpr int kUnroll = 4;
    const unsigned runs = capped(ceil_div_ll(blocks, kUnroll));
    if (aligned) {
      const dim3 grid(static_cast<unsigned>(ceil_div_ll(rows, kRowsPerCta)), runs);
      launch_dependent(quantize_fp8_rows_kernel, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    } else {
      const dim3 grid(static_cast<unsigned>(ceil_div_ll(rows, kThreads / 32)), runs);
      launch_dependent(quantize_fp8_odd_rows_kernel<kUnroll>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    }
    return launch_status();
  }
  const dim3 grid(static_cast<unsigned>(blocks), capped(ceil_div_ll(rows, kFp8Block)));
  if (aligned) launch_dependent(quantize_fp8_tiles_kernel, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  else launch_dependent(quantize_fp8_odd_tiles_kernel, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  return launch_status();
}

}  // namespace lc0b200
