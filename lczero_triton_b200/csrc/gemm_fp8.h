// Internal: the back ends behind lc0b200_gemm_fp8 / lc0b200_linear_fp8 (validated arguments only).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace lc0b200 {

struct GemmFp8 {
  void* out;
  const uint8_t* a;
  const float* a_scale;
  const uint8_t* w;
  const float* w_scale;
  const bf16* bias;
  long long m;
  int n, k;
  long long lda, ld_a_scale, ldw, ld_w_scale, ldc;
  int out_kind, activation;
};

// One value's activation.  A NaN stays one, and so does an infinity (mish(y) rounds to y above 20).
__device__ __forceinline__ float fp8_activate(float y, int activation) {
  if (activation == LC0B200_ACT_RELU) return y < 0.0f ? 0.0f : y;
  if (activation == LC0B200_ACT_MISH && y > 20.0f) return y;
  return activate_rt(y, activation);
}

// Chooses the kernel by what the operands allow.
int gemm_fp8(const GemmFp8& g, cudaStream_t stream);
// The dense layer on few bf16 rows in one launch (g.a, g.a_scale, g.lda and g.ld_a_scale are not used).
bool linear_fp8_few_supported(const GemmFp8& g, const bf16* a, long long lda);
int linear_fp8_few(const GemmFp8& g, const bf16* a, long long lda, cudaStream_t stream);
// CUDA-core kernel: any pitch and alignment.
int gemm_fp8_simt(const GemmFp8& g, cudaStream_t stream);

}  // namespace lc0b200
