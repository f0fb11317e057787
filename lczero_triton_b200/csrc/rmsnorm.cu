// Root-mean-square norm with the residual's addition in front of it and an e4m3 row behind it:
//   v = x + skip                     (f32; skip optional; bf16(v) may be stored as the new residual)
//   y = v / sqrt(mean(v^2) + eps) * gamma
//   out = bf16(y), and / or e4m3 codes with a scale per 1 x 128 block of the f32 y (fp8.cuh)
// Every result is rounded once, from the f32 value: the norm reads v and not the rounded residual, the codes come from
// y and not from the bf16 row, so that no result depends on which of the others are asked for.
// HBM-bound: a row is read once and kept in registers (rows of more than 16384 channels are read twice).
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace lc0b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarpsPerBlock = 2;  // rows per CTA of the one-warp kernels: more CTAs in flight, shorter tail

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
  int q_words;  // rows of codes start at multiples of 8 bytes
  float epsilon;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

__device__ __forceinline__ void unpack8(const uint4& raw, float (&f)[8]) {
  float2 t;
  t = unpack_bf16x2(raw.x); f[0] = t.x; f[1] = t.y;
  t = unpack_bf16x2(raw.y); f[2] = t.x; f[3] = t.y;
  t = unpack_bf16x2(raw.z); f[4] = t.x; f[5] = t.y;
  t = unpack_bf16x2(raw.w); f[6] = t.x; f[7] = t.y;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// Rows in registers as groups of eight channels, THREADS (32 or 256) threads a row: thread t holds groups t,
// t + THREADS, ...  Sixteen neighbouring lanes hold one 128-block of the e4m3 output.  SKIP, QUANT and the alignment of
// the rows are fixed at compile time, every load of the row is issued before any arithmetic.
template <int GROUPS, int THREADS, bool SKIP, bool QUANT, bool ALIGNED>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpsPerBlock : THREADS) rms_norm_kernel(const RmsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  // Group g of this thread starts at channel first + kStep g: a step of all threads, or, for rows that need shifting, of a
  // warp, which then walks a run of its own (store8_row).
  constexpr int kStep = 8 * (ALIGNED ? THREADS : 32);
  const int warp_in_row = THREADS == 32 ? 0 : threadIdx.x >> 5;
  const int warp_first = 256 * warp_in_row * (ALIGNED ? 1 : GROUPS);
  const int first = warp_first + 8 * lane;
  const long long row = THREADS == 32 ? blockIdx.x * static_cast<long long>(kWarpsPerBlock) + (threadIdx.x >> 5) : blockIdx.x;
  if (THREADS == 32 && row >= p.rows) return;
  const bf16* x = p.x + row * p.ld_x;
  const bf16* skip = p.skip + row * p.ld_skip;
  const bool inner = inner_row(row, p.rows, p.ld_x), inner_skip = SKIP && inner_row(row, p.rows, p.ld_skip);
  RowWords raw[GROUPS], raw_skip[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    raw[g] = load_words<ALIGNED>(x, first + kStep * g, p.width, inner);
    if (SKIP) raw_skip[g] = load_words<ALIGNED>(skip, first + kStep * g, p.width, inner_skip);
  }
  float v[GROUPS][8];  // zeros past the row's end
  float sum = 0.0f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int col = first + kStep * g;
    unpack8(channels_of<ALIGNED>(raw[g], x, col, p.width), v[g]);
    if (SKIP) {
      float s[8];
      unpack8(channels_of<ALIGNED>(raw_skip[g], skip, col, p.width), s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] += s[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(v[g][j], v[g][j], sum);
  }
  sum = warp_sum(sum);
  if (THREADS > 32) {
    __shared__ float warp_part[THREADS / 32];
    if (lane == 0) warp_part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) sum += warp_part[w];
  }
  __syncwarp();
  // Every thread of the row has its operands from here on (a lane may have read a word that holds its neighbour's channels):
  // results may lie over them.
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.width) + p.epsilon);
  const bool gamma_words = ALIGNED || aligned16_dev(p.gamma);
  uint4 carry_residual = make_uint4(0u, 0u, 0u, 0u), carry_out = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    if (warp_first + kStep * g >= p.width) break;  // the same for the warp: the shuffles below have every lane
    const int col = first + kStep * g;
    const bool begin = g == 0, end = g + 1 == GROUPS;
    if (SKIP && p.residual != nullptr) store8_row<ALIGNED>(p.residual + row * p.ld_residual, col, p.width, pack8(v[g]), carry_residual, begin, end);
    uint4 gamma_raw = make_uint4(0u, 0u, 0u, 0u);
    if (gamma_words && col + 8 <= p.width) gamma_raw = __ldg(reinterpret_cast<const uint4*>(p.gamma + col));
    else if (!ALIGNED && col < p.width) gamma_raw = edge_word(p.gamma, col, p.width);
    float gamma[8];
    unpack8(gamma_raw, gamma);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[g][j] = v[g][j] * rstd * gamma[j];
    if (col + 8 > p.width) {  // (0 * rstd may be NaN, and these channels share a block's maximum)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] = col + j < p.width ? v[g][j] : 0.0f;
    }
    if (p.out != nullptr) store8_row<ALIGNED>(p.out + row * p.ld_out, col, p.width, pack8(v[g]), carry_out, begin, end);
    if (QUANT) {
      uint32_t amax = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = max(amax, magnitude_bits(v[g][j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
      float scale, inverse;
      fp8_block_scale(amax, scale, inverse);
      if (col < p.width) {
        if ((lane & 15) == 0) p.scale[(col / kFp8Block) * p.ld_scale + row] = scale;
        const uint32_t lo = fp8_pack4(v[g][0] * inverse, v[g][1] * inverse, v[g][2] * inverse, v[g][3] * inverse);
        const uint32_t hi = fp8_pack4(v[g][4] * inverse, v[g][5] * inverse, v[g][6] * inverse, v[g][7] * inverse);
        uint8_t* q = p.q + row * p.ld_q + col;
        if (ALIGNED || (p.q_words && col + 8 <= p.width)) {
          *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (col + j < p.width) q[j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
          }
        }
      }
    }
  }
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

template <int GROUPS, int THREADS, bool ALIGNED>
void launch_rows(const RmsParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(THREADS == 32 ? ceil_div_ll(p.rows, kWarpsPerBlock) : p.rows));
  const dim3 block(THREADS == 32 ? 32 * kWarpsPerBlock : THREADS);
  const bool skip = p.skip != nullptr, quant = p.q != nullptr;
  if (skip && quant) launch_dependent(rms_norm_kernel<GROUPS, THREADS, true, true, ALIGNED>, grid, block, 0, st, p);
  else if (skip) launch_dependent(rms_norm_kernel<GROUPS, THREADS, true, false, ALIGNED>, grid, block, 0, st, p);
  else if (quant) launch_dependent(rms_norm_kernel<GROUPS, THREADS, false, true, ALIGNED>, grid, block, 0, st, p);
  else launch_dependent(rms_norm_kernel<GROUPS, THREADS, false, false, ALIGNED>, grid, block, 0, st, p);
}

template <bool ALIGNED>
bool launch_held(const RmsParams& p, cudaStream_t st) {
  // One warp per row up to 2048 channels, but not where there are fewer rows than SMs: a CTA then shares the row out.
  const int width = p.width;
  if (width <= 2048 && (p.rows > sm_count() || width <= 256)) {
    if (width <= 256) launch_rows<1, 32, ALIGNED>(p, st);
    else if (width <= 512) launch_rows<2, 32, ALIGNED>(p, st);
    else if (width <= 1024) launch_rows<4, 32, ALIGNED>(p, st);
    else if (width <= 1536) launch_rows<6, 32, ALIGNED>(p, st);
    else launch_rows<8, 32, ALIGNED>(p, st);
    return true;
  }
  if (width <= 2048) launch_rows<1, 256, ALIGNED>(p, st);
  else if (width <= 4096) launch_rows<2, 256, ALIGNED>(p, st);
  else if (width <= 8192) launch_rows<4, 256, ALIGNED>(p, st);
  else if (width <= 16384) launch_rows<8, 256, ALIGNED>(p, st);
  else return false;
  return true;
}

// 16-byte accesses to every row of a bf16 operand that is there.
bool rows_aligned16(const void* base, long long ld) { return base == nullptr || (aligned16(base) && (ld % 8) == 0); }

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
  p.q_words = (reinterpret_cast<uintptr_t>(q_out) % 8) == 0 && (ld_q % 8) == 0;
  const bool aligned = (width % 8) == 0 && rows_aligned16(in, ld_in) && rows_aligned16(skip, ld_skip) && rows_aligned16(out, ld_out) &&
                       rows_aligned16(residual, ld_residual) && aligned16(gamma) && p.q_words;
  if (aligned ? launch_held<true>(p, st) : launch_held<false>(p, st)) return launch_status();
  launch_dependent(rms_norm_any_kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st, p);
  return launch_status();
}

}  // namespace lc0b200
