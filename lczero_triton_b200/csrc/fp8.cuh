// The e4m3 block rule shared by the kernels that produce 8-bit floating rows.
//
// Block of 128 values (1 x 128 for activations, 128 x 128 for weights):
//   amax  = max |x|                          a NaN stays a NaN, an infinity stays one
//   scale = amax / 448                       1 where amax < 2^-117: such a block counts as zeros
//   code  = e4m3(x * (448 / amax))           IEEE division once per block, round half to even, saturated to +-448
// 2^-117 is where 448 / amax still is a finite float (it overflows below 2^-119.2).  Non-finite blocks cannot hide:
// amax = inf gives scale = inf and codes 0 and NaN, amax = NaN gives scale = NaN, so every value of such a block
// reads back as NaN.
#pragma once

#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

namespace lc0b200 {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.0f;
constexpr uint32_t kFp8TinyBits = 0x05000000u;  // 2^-117 as float bits

// Sixteen lanes hold four blocks: the maxima of all four reduced together, each exchange halving what a lane still carries;
// lane l (of sixteen) ends with block l / 4's.  Five shuffles instead of sixteen, and what follows (two or three IEEE
// divisions a block) is done once a lane instead of four times.
__device__ __forceinline__ uint32_t max_of_four_blocks(const uint32_t (&m)[4]) {
  const bool upper = (threadIdx.x & 8) != 0, odd = (threadIdx.x & 4) != 0;
  const uint32_t s0 = __shfl_xor_sync(0xFFFFFFFFu, upper ? m[0] : m[2], 8), s1 = __shfl_xor_sync(0xFFFFFFFFu, upper ? m[1] : m[3], 8);
  const uint32_t k0 = max(upper ? m[2] : m[0], s0), k1 = max(upper ? m[3] : m[1], s1);
  uint32_t k = max(odd ? k1 : k0, __shfl_xor_sync(0xFFFFFFFFu, odd ? k0 : k1, 4));
  k = max(k, __shfl_xor_sync(0xFFFFFFFFu, k, 2));
  return max(k, __shfl_xor_sync(0xFFFFFFFFu, k, 1));
}
// Block u's value of the four, from the lanes that hold it.
template <typename T>
__device__ __forceinline__ T from_block(T value, int u) {
  return __shfl_sync(0xFFFFFFFFu, value, (threadIdx.x & 16) + 4 * u);
}

// |x| as bits: unsigned order is the order of magnitudes with every NaN above infinity, so an integer maximum keeps NaN.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ void fp8_block_scale(uint32_t amax_bits, float& scale, float& inverse) {
  const float amax = __uint_as_float(amax_bits);
  const bool zeros = amax_bits < kFp8TinyBits;
  scale = zeros ? 1.0f : __fdiv_rn(amax, kFp8Max);
  inverse = zeros ? 1.0f : __fdiv_rn(kFp8Max, amax);
}

// The same for a block of y = t * rstd, from the maximum of |t|: the factor 448 / max|t| gives the codes from t itself, two
// roundings instead of four.  False where that is not safe (a factor that overflows, zeros, a row that is not finite):
// then `factor` is for y.
__device__ __forceinline__ bool fp8_norm_block_scale(uint32_t amax_bits, float rstd, float& scale, float& factor) {
  const float amax = __uint_as_float(amax_bits), amax_y = amax * rstd;
  fp8_block_scale(magnitude_bits(amax_y), scale, factor);
  const bool direct = amax_bits >= kFp8TinyBits && amax_y >= __uint_as_float(kFp8TinyBits) && amax_y <= 3.0e38f && amax <= 3.0e38f;
  if (direct) factor = __fdiv_rn(kFp8Max, amax);
  return direct;
}

__device__ __forceinline__ uint16_t fp8_pack2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

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

__device__ __forceinline__ float fp8_value(uint8_t code) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(code, __NV_E4M3);
  return __half2float(__half(h));
}

}  // namespace lc0b200
