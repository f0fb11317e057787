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

__device__ __forceinline__ uint2 codes8(const uint4& raw, float inverse) {
  const float2 a = unpack_bf16x2(raw.x), b = unpack_bf16x2(raw.y), c = unpack_bf16x2(raw.z), d = unpack_bf16x2(raw.w);
  return make_uint2(fp8_pack4(a.x * inverse, a.y * inverse, b.x * inverse, b.y * inverse),
                    fp8_pack4(c.x * inverse, c.y * inverse, d.x * inverse, d.y * inverse));
}

// Rows of whole, aligned 16-byte words: a half-warp takes UNROLL neighbouring blocks of one row, a CTA 16 rows.
template <int UNROLL>
__global__ void __launch_bounds__(kThreads)
quantize_fp8_rows_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                         int width, long long ld_in, long long ld_out, long long ld_scale) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane16 = threadIdx.x & 15;
  const long long row = blockIdx.x * static_cast<long long>(kRowsPerCta) + (threadIdx.x >> 4);
  const int groups = row < rows ? width >> 3 : 0;  // a half-warp without a row stays for the other half's shuffles
  const uint4* src = reinterpret_cast<const uint4*>(x + row * ld_in);
  uint2* dst = reinterpret_cast<uint2*>(q_out + row * ld_out);
  const int blocks = static_cast<int>(ceil_div_ll(width, kFp8Block));
  for (int first = blockIdx.y * UNROLL; first < blocks; first += gridDim.y * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int idx = (first + u) * 16 + lane16;
      raw[u] = idx < groups ? __ldg(src + idx) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int idx = (first + u) * 16 + lane16;
      uint32_t m = packed_magnitude(raw[u]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      float scale, inverse;
      fp8_block_scale(magnitude_of_packed(m), scale, inverse);
      if (idx < groups) {
        if (lane16 == 0) scale_out[(first + u) * ld_scale + row] = scale;
        dst[idx] = codes8(raw[u], inverse);
      }
    }
  }
}

// Rows of any alignment and width, pairs of channels a lane (rows.cuh): a warp takes UNROLL neighbouring blocks of a row.
template <int UNROLL>
__global__ void __launch_bounds__(kThreads)
quantize_fp8_row_pairs_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                              int width, long long ld_in, long long ld_out, long long ld_scale, bool even) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.x * static_cast<long long>(kThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const bf16* src = x + row * ld_in;
  const int half = row_half(src);
  const bool inner = inner_row(row, rows, ld_in);
  for (long long run = blockIdx.y * static_cast<long long>(UNROLL * kFp8Block); run < width; run += gridDim.y * static_cast<long long>(UNROLL * kFp8Block)) {
    uint32_t w[2 * UNROLL + 1];
    load_row_words<2 * UNROLL>(w, src, static_cast<int>(run), width, inner);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int c = static_cast<int>(run) + kFp8Block * u + 2 * lane;
      if (c - 2 * lane >= width) break;  // the same for the warp
      uint32_t pair[2] = {row_pair<2 * UNROLL>(w, 2 * u, half), row_pair<2 * UNROLL>(w, 2 * u + 1, half)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (c + 64 * i + 1 >= width) pair[i] = c + 64 * i < width ? pair[i] & 0xFFFFu : 0u;
      }
      const uint32_t m = __vmaxu2(pair[0] & 0x7FFF7FFFu, pair[1] & 0x7FFF7FFFu);
      float scale, inverse;
      fp8_block_scale(__reduce_max_sync(0xFFFFFFFFu, magnitude_of_packed(m)), scale, inverse);
      if (lane == 0) scale_out[(c / kFp8Block) * ld_scale + row] = scale;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 v = unpack_bf16x2(pair[i]);
        store_code_pair(q_out + row * ld_out, c + 64 * i, width, even, v.x * inverse, v.y * inverse);
      }
    }
  }
}

// The maximum over a CTA's threads of magnitude bits.  `words` (one per warp) is used for every other tile only, so that the
// next tile's writes cannot overtake this tile's reads.
__device__ __forceinline__ uint32_t cta_max(uint32_t m, uint32_t* words) {
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max(m, words[w]);
  return m;
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

// ... and for rows of any alignment and width: a warp holds sixteen rows of the tile, two steps of pairs each.
__global__ void __launch_bounds__(kThreads)
quantize_fp8_tile_pairs_kernel(uint8_t* __restrict__ q_out, float* __restrict__ scale_out, const bf16* __restrict__ x, long long rows,
                               int width, long long ld_in, long long ld_out, long long ld_scale, bool even) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ uint32_t warp_max[2][kThreads / 32];
  constexpr int kRowsPerWarp = kFp8Block / (kThreads / 32);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = blockIdx.x * kFp8Block;
  const long long row_tiles = ceil_div_ll(rows, kFp8Block);
  int parity = 0;
  for (long long tile = blockIdx.y; tile < row_tiles; tile += gridDim.y, parity ^= 1) {
    const long long row0 = tile * kFp8Block + warp;  // then every eighth
    uint32_t w[kRowsPerWarp][3];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      const long long row = row0 + 8 * i;
      w[i][0] = w[i][1] = w[i][2] = 0u;
      if (row < rows) load_row_words<2>(w[i], x + row * ld_in, run, width, inner_row(row, rows, ld_in));
    }
    uint32_t m = 0u, pair[kRowsPerWarp][2];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int c = run + 64 * s + 2 * lane;
        pair[i][s] = row_pair<2>(w[i], s, row_half(x + (row0 + 8 * i) * ld_in));
        if (c + 1 >= width) pair[i][s] = c < width ? pair[i][s] & 0xFFFFu : 0u;
        m = __vmaxu2(m, pair[i][s] & 0x7FFF7FFFu);
      }
    }
    float scale, inverse;
    fp8_block_scale(cta_max(magnitude_of_packed(m), warp_max[parity]), scale, inverse);
    if (threadIdx.x == 0) scale_out[tile * ld_scale + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      const long long row = row0 + 8 * i;
      if (row < rows) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float2 v = unpack_bf16x2(pair[i][s]);
          store_code_pair(q_out + row * ld_out, run + 64 * s + 2 * lane, width, even, v.x * inverse, v.y * inverse);
        }
      }
    }
  }
}

}  // namespace

int quantize_fp8(void* out, float* scale, const void* in, long long rows, int width, int block_rows, long long ld_in,
                 long long ld_out, long long ld_scale, cudaStream_t st) {
  auto* q = reinterpret_cast<uint8_t*>(out);
  const auto* x = reinterpret_cast<const bf16*>(in);
  const bool aligned = (width % 8) == 0 && aligned16(in) && (ld_in % 8) == 0 && (reinterpret_cast<uintptr_t>(out) % 8) == 0 && (ld_out % 8) == 0;
  const bool even = ((reinterpret_cast<uintptr_t>(out) | static_cast<unsigned long long>(ld_out)) & 1u) == 0;
  const long long blocks = ceil_div_ll(width, kFp8Block);
  const dim3 threads(kThreads);
  auto capped = [](long long count) { return static_cast<unsigned>(count < 65535 ? count : 65535); };
  if (block_rows == 1) {
    constexpr int kUnroll = 4;
    const unsigned runs = capped(ceil_div_ll(blocks, kUnroll));
    if (aligned) {
      const dim3 grid(static_cast<unsigned>(ceil_div_ll(rows, kRowsPerCta)), runs);
      launch_dependent(quantize_fp8_rows_kernel<kUnroll>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
    } else {
      const dim3 grid(static_cast<unsigned>(ceil_div_ll(rows, kThreads / 32)), runs);
      launch_dependent(quantize_fp8_row_pairs_kernel<kUnroll>, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale, even);
    }
    return launch_status();
  }
  const dim3 grid(static_cast<unsigned>(blocks), capped(ceil_div_ll(rows, kFp8Block)));
  if (aligned) launch_dependent(quantize_fp8_tiles_kernel, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale);
  else launch_dependent(quantize_fp8_tile_pairs_kernel, grid, threads, 0, st, q, scale, x, rows, width, ld_in, ld_out, ld_scale, even);
  return launch_status();
}

}  // namespace lc0b200
