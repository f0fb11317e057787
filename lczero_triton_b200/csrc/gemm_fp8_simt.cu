// CUDA-core form of the block-scaled e4m3 product, for operands TMA cannot address (a base or a row pitch that is not a
// multiple of 16 bytes) and as an independent cross-check of the tensor-core kernels.  64 x 64 output tile per CTA,
// 4 x 4 per thread, bound by the fp32 pipes and shared memory, and for few rows by one CTA's walk along k: 8192 x 1024 x 1001 in
// 792 us (21 TFLOP/s; in brackets the time with a pitch that TMA takes: 16), 777 x 1858 x 1001 in 244 (9), 64 x 1536 x 1001 in
// 107 (5), 1 x 4096 x 4095 in 352 (6).  As in them, a block's sum is formed from the codes and then
// multiplied by the product of its two scales.
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "gemm_fp8.h"

namespace lc0b200 {

namespace {

constexpr int kTile = 64;
constexpr int kTileK = 16;
constexpr int kMaxGridY = 65535;
static_assert(kFp8Block % kTileK == 0 && kFp8Block % kTile == 0, "a step along k, or a tile, must not straddle two scales");

// MANY: more tiles of columns than a grid has in y; they continue in z.  (A kernel of its own: with these two lines every
// product took 2 to 15 % longer, with a loop over the tiles 20 to 45 %.)
template <bool MANY>
__global__ void __launch_bounds__(256) gemm_fp8_simt_kernel(const GemmFp8 p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float sa[kTileK][kTile + 1];
  __shared__ float sw[kTileK][kTile + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long m0 = static_cast<long long>(blockIdx.x) * kTile;
  const int n0 = (MANY ? blockIdx.z * kMaxGridY + blockIdx.y : blockIdx.y) * kTile;
  if (MANY && n0 >= p.n) return;
  float acc[4][4] = {}, block[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTile * kTileK; i += 256) {
      const int r = i / kTileK, c = i % kTileK;
      const long long gm = m0 + r;
      const int gn = n0 + r, gk = k0 + c;
      sa[c][r] = (gm < p.m && gk < p.k) ? fp8_value(p.a[gm * p.lda + gk]) : 0.0f;
      sw[c][r] = (gn < p.n && gk < p.k) ? fp8_value(p.w[gn * p.ldw + gk]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kTileK; ++kk) {
      float av[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = sa[kk][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) wv[j] = sw[kk][tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) block[i][j] = fmaf(av[i], wv[j], block[i][j]);
      }
    }
    if (k0 + kTileK >= p.k || (k0 + kTileK) % kFp8Block == 0) {
      const int kb = k0 / kFp8Block;
      const float w_scale = p.w_scale[(n0 / kFp8Block) * p.ld_w_scale + kb];  // a tile lies in one row of scales
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long gm = m0 + ty * 4 + i;
        const float scale = gm < p.m ? p.a_scale[kb * p.ld_a_scale + gm] * w_scale : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(block[i][j], scale, acc[i][j]);
          block[i][j] = 0.0f;
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long gm = m0 + ty * 4 + i;
    if (gm >= p.m) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int gn = n0 + tx * 4 + j;
      if (gn >= p.n) continue;
      float y = acc[i][j] + (p.bias != nullptr ? __bfloat162float(p.bias[gn]) : 0.0f);
      y = fp8_activate(y, p.activation);
      if (p.out_kind == LC0B200_OUT_F32) reinterpret_cast<float*>(p.out)[gm * p.ldc + gn] = y;
      else reinterpret_cast<bf16*>(p.out)[gm * p.ldc + gn] = __float2bfloat16_rn(y);
    }
  }
}

}  // namespace

int gemm_fp8_simt(const GemmFp8& g, cudaStream_t stream) {
  const long long n_tiles = ceil_div_ll(g.n, kTile);
  const dim3 grid(static_cast<unsigned>(ceil_div_ll(g.m, kTile)), static_cast<unsigned>(n_tiles < kMaxGridY ? n_tiles : kMaxGridY),
                  static_cast<unsigned>(ceil_div_ll(n_tiles, kMaxGridY)));
  if (grid.z > 1) launch_dependent(gemm_fp8_simt_kernel<true>, grid, dim3(256), 0, stream, g);
  else launch_dependent(gemm_fp8_simt_kernel<false>, grid, dim3(256), 0, stream, g);
  return launch_status();
}

}  // namespace lc0b200
