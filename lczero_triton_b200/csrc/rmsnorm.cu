// Root-mean-square norm with the residual's addition in front of it and an e4m3 row behind it:
//   v = x + skip                     (f32; skip optional; bf16(v) may be stored as the new residual)
//   y = v / sqrt(mean(v^2) + eps) * gamma
//   out = bf16(y), and / or e4m3 codes with a scale per 1 x 128 block of the f32 y (fp8.cuh)
// Every result is rounded once, from the f32 value: the norm reads v and not the rounded residual, the codes come from
// y and not from the bf16 row, so that no result depends on which of the others are asked for.
// HBM-bound: each row is read once and kept on chip.
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace lc0b200 {

namespace {

constexpr int kThreads = 256;

struct RmsParams {
  bf16* out;
  bf16* residual;
  uint8_t* q;
  float* scale;
  const bf16* x;
  const bf16* skip;
  const bf16* gamma;
  long long rows, ld_x, ld_skip, ld_out, ld_residual, ld_q, ld_scale;
  int width;
  float epsilon;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Any width, pitch and alignment: one CTA per row, the row read twice (the second time from the caches).  Every value
// is read and written by the same thread in the second pass only, so results may lie over their inputs.
__global__ void __launch_bounds__(kThreads) rms_norm_any_kernel(const RmsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float warp_part[kThreads / 32];
  const long long row = blockIdx.x;
  const bf16* x = p.x + row * p.ld_x;
  const bf16* skip = p.skip != nullptr ? p.skip + row * p.ld_skip : nullptr;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto value = [&](int c) {
    const float v = __bfloat162float(x[c]);
    return skip != nullptr ? v + __bfloat162float(skip[c]) : v;
  };
  float sum = 0.0f;
  for (int c = threadIdx.x; c < p.width; c += kThreads) {
    const float v = value(c);
    sum = fmaf(v, v, sum);
  }
  sum = warp_sum(sum);
  if (lane == 0) warp_part[warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += warp_part[w];
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.width) + p.epsilon);
  // A warp takes whole 128-blocks, four values a lane.
  const int blocks = static_cast<int>(ceil_div_ll(p.width, kFp8Block));
  for (int block = warp; block < blocks; block += kThreads / 32) {
    float y[4];
    uint32_t amax = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = block * kFp8Block + 32 * j + lane;
      y[j] = 0.0f;
      if (c < p.width) {
        const float v = value(c);
        y[j] = v * rstd * __bfloat162float(p.gamma[c]);
        if (p.residual != nullptr) p.residual[row * p.ld_residual + c] = __float2bfloat16_rn(v);
        if (p.out != nullptr) p.out[row * p.ld_out + c] = __float2bfloat16_rn(y[j]);
      }
      amax = max(amax, magnitude_bits(y[j]));
    }
    if (p.q != nullptr) {
      float scale, inverse;
      fp8_block_scale(__reduce_max_sync(0xFFFFFFFFu, amax), scale, inverse);
      if (lane == 0) p.scale[block * p.ld_scale + row] = scale;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = block * kFp8Block + 32 * j + lane;
        if (c < p.width) p.q[row * p.ld_q + c] = fp8_one(y[j] * inverse);
      }
    }
  }
}

}  // namespace

int rms_norm(void* out, void* residual, void* q_out, float* q_scale, const void* in, const void* skip, const void* gamma,
             long long rows, int width, float epsilon, long long ld_in, long long ld_skip, long long ld_out,
             long long ld_residual, long long ld_q, long long ld_scale, cudaStream_t st) {
  RmsParams p;
  p.out = reinterpret_cast<bf16*>(out);
  p.residual = reinterpret_cast<bf16*>(residual);
  p.q = reinterpret_cast<uint8_t*>(q_out);
  p.scale = q_scale;
  p.x = reinterpret_cast<const bf16*>(in);
  p.skip = reinterpret_cast<const bf16*>(skip);
  p.gamma = reinterpret_cast<const bf16*>(gamma);
  p.rows = rows;
  p.ld_x = ld_in;
  p.ld_skip = ld_skip;
  p.ld_out = ld_out;
  p.ld_residual = ld_residual;
  p.ld_q = ld_q;
  p.ld_scale = ld_scale;
  p.width = width;
  p.epsilon = epsilon;
  launch_dependent(rms_norm_any_kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st, p);
  return launch_status();
}

}  // namespace lc0b200
