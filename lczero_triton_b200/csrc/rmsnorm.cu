// Root-mean-square norm with the residual's addition in front of it and an e4m3 row behind it:
//   v = x + skip                     (f32; skip optional; bf16(v) may be stored as the new residual)
//   y = v / sqrt(mean(v^2) + eps) * gamma
//   out = bf16(y), and / or e4m3 codes with a scale per 1 x 128 block of the f32 y (fp8.cuh)
// Every result is rounded once, from the f32 value: the norm reads v and not the rounded residual, the codes come from
// y and not from the bf16 row, so that no result depends on which of the others are asked for.  y = (v * gamma) * rstd:
// without a skip v * gamma is a product of two bf16 values and exact (with one, v is an f32 sum and the product rounds), and as
// rstd is a factor of the whole row, the codes come from v * gamma alone.
// HBM-bound: a row is read once and kept in registers (rows of more than 16384 channels are read twice, a channel an access
// whatever their alignment: 2048 x 20480 with skip and residual in 147 us, 2.3 TB/s, where 16384 channels take 47).  262144 x 1024 with
// skip, residual, bf16 and codes: 360 us, 6.8 TB/s.  One row of 4096: 1.9 us, latency.  Rows of any alignment are bound by
// the number of memory instructions: 5003 x 1111 with skip and residual in 11.3 us, its bytes take 6.8.
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"

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
  float epsilon;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sum over the 16, 32 or 256 threads of a row.
template <int THREADS>
__device__ __forceinline__ float row_sum(float sum) {
#pragma unroll
  for (int o = THREADS < 32 ? THREADS / 2 : 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (THREADS <= 32) return sum;
  __shared__ float warp_part[THREADS < 32 ? 1 : THREADS / 32];
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) sum += warp_part[w];
  return sum;
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

// Rows in registers as 16-byte groups of eight channels, THREADS (16, 32 or 256) threads a row: thread t holds groups t,
// t + THREADS, ...  Sixteen neighbouring lanes hold one 128-block of the e4m3 output.  SKIP and QUANT are fixed at compile
// time, every load of the row is issued before any arithmetic.
template <int GROUPS, int THREADS, bool SKIP, bool QUANT>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpsPerBlock : 256) rms_norm_kernel(const RmsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int t = threadIdx.x % THREADS;
  const long long row = blockIdx.x * static_cast<long long>(blockDim.x / THREADS) + threadIdx.x / THREADS;
  if (THREADS == 32 && row >= p.rows) return;
  const int groups = row < p.rows ? p.width >> 3 : 0;  // a half-warp without a row stays for the other half's shuffles
  const uint4* x = reinterpret_cast<const uint4*>(p.x + row * p.ld_x);
  const uint4* skip = reinterpret_cast<const uint4*>(p.skip + row * p.ld_skip);
  uint4 raw[GROUPS], raw_skip[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int idx = t + THREADS * g;
    raw[g] = raw_skip[g] = make_uint4(0u, 0u, 0u, 0u);
    if (idx < groups) {
      raw[g] = x[idx];
      if (SKIP) raw_skip[g] = skip[idx];
    }
  }
  // A CTA per row is for few or wide rows, where a second memory round trip shows: gamma comes with the row.
  constexpr bool kGammaEarly = THREADS == 256 && GROUPS <= 4;
  uint4 raw_gamma[GROUPS];
  if (kGammaEarly) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (t + THREADS * g < groups) raw_gamma[g] = __ldg(reinterpret_cast<const uint4*>(p.gamma) + t + THREADS * g);
    }
  }
  float v[GROUPS][8];
  float sum = 0.0f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    unpack8(raw[g], v[g]);
    if (SKIP) {
      float s[8];
      unpack8(raw_skip[g], s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] += s[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(v[g][j], v[g][j], sum);
  }
  sum = row_sum<THREADS>(sum);
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.width) + p.epsilon);
  if (SKIP && p.residual != nullptr) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int idx = t + THREADS * g;
      if (idx < groups) reinterpret_cast<uint4*>(p.residual + row * p.ld_residual)[idx] = pack8(v[g]);
    }
  }
  if (rstd == 0.0f) {  // the squares overflowed: zeros, whatever gamma is (an infinity gives NaN)
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] *= 0.0f;
    }
  }
#pragma unroll
  for (int g0 = 0; g0 < GROUPS; g0 += 4) {
    if (THREADS * g0 >= (p.width >> 3)) break;  // the same for every row: the shuffles below have every lane
    uint32_t amax[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int g = g0; g < GROUPS && g < g0 + 4; ++g) {
      const int idx = t + THREADS * g;
      if (idx >= groups) continue;
      float gamma[8], y[8];
      unpack8(kGammaEarly ? raw_gamma[g] : __ldg(reinterpret_cast<const uint4*>(p.gamma) + idx), gamma);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[g][j] *= gamma[j];
        y[j] = v[g][j] * rstd;
        if (QUANT) amax[g - g0] = max(amax[g - g0], magnitude_bits(v[g][j]));
      }
      if (p.out != nullptr) reinterpret_cast<uint4*>(p.out + row * p.ld_out)[idx] = pack8(y);
    }
    if (QUANT) {
      // Sixteen lanes hold block (t + THREADS g) / 16 in step g: four steps at a time, a lane works out one block's scale.
      float scale, factor;
      const bool direct = fp8_norm_block_scale(max_of_four_blocks(amax), rstd, scale, factor);
      const int step = g0 + ((lane >> 2) & 3), block = ((t & ~15) + THREADS * step) / 16;
      if ((lane & 3) == 0 && step < GROUPS && row < p.rows && block * 16 < groups) p.scale[block * p.ld_scale + row] = scale;
      const float before = direct ? 1.0f : rstd;
#pragma unroll
      for (int g = g0; g < GROUPS && g < g0 + 4; ++g) {
        const int idx = t + THREADS * g;
        const float f = from_block(factor, g - g0), r = from_block(before, g - g0);
        if (r != 1.0f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[g][j] *= r;
        }
        if (idx < groups) {
          reinterpret_cast<uint2*>(p.q + row * p.ld_q)[idx] = make_uint2(fp8_pack4(v[g][0] * f, v[g][1] * f, v[g][2] * f, v[g][3] * f),
                                                                        fp8_pack4(v[g][4] * f, v[g][5] * f, v[g][6] * f, v[g][7] * f));
        }
      }
    }
  }
}

// Rows of any alignment and width: a warp takes a run of 32 CHANNELS channels, channel run + lane + 32 i to a lane, so that
// a warp's access is one run of memory and four channels of a lane make a 128-block; as many warps a row as it has runs.
// Eight channels a lane keep many rows in flight: with a whole row of 1111 to a warp (48 channels a lane, 137 registers) 5003
// rows took 27 us.  (16-byte or 4-byte words shifted into place move fewer requests and execute three times the instructions: 26 and
// 37 us, with a whole row to a warp; with eight channels a lane they were not tried.)
// FULL: the run lies inside the row, nothing is checked per channel.
template <int CHANNELS, bool SKIP, bool FULL>
__device__ __forceinline__ float load_run(const RmsParams& p, long long row, int c0, float (&v)[CHANNELS], bf16 (&gamma)[CHANNELS]) {
  const bf16* x = p.x + row * p.ld_x + c0;
  const bf16* skip = p.skip + row * p.ld_skip + c0;
  bf16 raw[CHANNELS], raw_skip[CHANNELS];
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i) {
    raw[i] = raw_skip[i] = gamma[i] = __ushort_as_bfloat16(0);
    if (FULL || c0 + 32 * i < p.width) {
      raw[i] = x[32 * i];
      if (SKIP) raw_skip[i] = skip[32 * i];
      gamma[i] = p.gamma[c0 + 32 * i];  // here already: one memory round trip a row, not two
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i) {
    v[i] = __bfloat162float(raw[i]);
    if (SKIP) v[i] += __bfloat162float(raw_skip[i]);
    sum = fmaf(v[i], v[i], sum);
  }
  return sum;
}

template <int CHANNELS, bool SKIP, bool QUANT, bool FULL>
__device__ __forceinline__ void store_run(const RmsParams& p, long long row, int c0, float (&v)[CHANNELS], const bf16 (&gamma)[CHANNELS], float rstd) {
  bf16* residual = p.residual + row * p.ld_residual + c0;
  bf16* out = p.out + row * p.ld_out + c0;
  if (SKIP && p.residual != nullptr) {
#pragma unroll
    for (int i = 0; i < CHANNELS; ++i) {
      if (FULL || c0 + 32 * i < p.width) residual[32 * i] = __float2bfloat16_rn(v[i]);
    }
  }
  if (rstd == 0.0f) {  // the squares overflowed: zeros, whatever gamma is (an infinity gives NaN)
#pragma unroll
    for (int i = 0; i < CHANNELS; ++i) v[i] *= 0.0f;
  }
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i) {
    const bool here = FULL || c0 + 32 * i < p.width;
    v[i] *= __bfloat162float(gamma[i]);  // (both zero past the row's end)
    if (p.out != nullptr && here) out[32 * i] = __float2bfloat16_rn(v[i] * rstd);
  }
  if (QUANT) {
    uint8_t* q = p.q + row * p.ld_q + c0;
    const int lane = threadIdx.x & 31, block0 = (c0 - lane) / kFp8Block;
    // Lane u works out block u's scale (three divisions once, not CHANNELS / 4 times).
    uint32_t mine = 0u;
#pragma unroll
    for (int u = 0; u < CHANNELS / 4; ++u) {
      uint32_t amax = 0u;
#pragma unroll
      for (int i = 4 * u; i < 4 * u + 4; ++i) amax = max(amax, magnitude_bits(v[i]));
      amax = __reduce_max_sync(0xFFFFFFFFu, amax);
      mine = lane == u ? amax : mine;
    }
    float scale, factor;
    const bool direct = fp8_norm_block_scale(mine, rstd, scale, factor);
    if (lane < CHANNELS / 4 && (FULL || (block0 + lane) * kFp8Block < p.width)) p.scale[(block0 + lane) * p.ld_scale + row] = scale;
#pragma unroll
    for (int u = 0; u < CHANNELS / 4; ++u) {
      const float f = __shfl_sync(0xFFFFFFFFu, factor, u), r = __shfl_sync(0xFFFFFFFFu, direct ? 1.0f : rstd, u);
#pragma unroll
      for (int i = 4 * u; i < 4 * u + 4; i += 2) {
        const uint16_t codes = r == 1.0f ? fp8_pack2(v[i] * f, v[i + 1] * f) : fp8_pack2(v[i] * r * f, v[i + 1] * r * f);
        if (FULL || c0 + 32 * i < p.width) q[32 * i] = static_cast<uint8_t>(codes);
        if (FULL || c0 + 32 * i + 32 < p.width) q[32 * i + 32] = static_cast<uint8_t>(codes >> 8);
      }
    }
  }
}

// MANY: blockDim.y narrow rows a CTA.  With a CTA for every row the kernel is bound by how fast CTAs start (100000 rows of 61:
// 104 us, 52 so); for rows of more than two warps one row is the faster (20000 x 1001: 43 us, 47 with two).
template <int CHANNELS, bool SKIP, bool QUANT, bool MANY>
__global__ void __launch_bounds__(1024) rms_norm_odd_kernel(const RmsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float warp_part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long row = MANY ? blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y : blockIdx.x;
  const bool here = !MANY || row < p.rows;
  const int c0 = 32 * CHANNELS * warp + lane;
  const bool full = 32 * CHANNELS * (warp + 1) <= p.width;
  float v[CHANNELS];
  bf16 gamma[CHANNELS];
  float sum = 0.0f;
  if (here) sum = warp_sum(full ? load_run<CHANNELS, SKIP, true>(p, row, c0, v, gamma) : load_run<CHANNELS, SKIP, false>(p, row, c0, v, gamma));
  if (warps > 1) {
    float* part = MANY ? warp_part + threadIdx.y * warps : warp_part;
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = warp_sum(lane < warps ? part[lane] : 0.0f);
  }
  if (!here) return;
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.width) + p.epsilon);
  if (full) store_run<CHANNELS, SKIP, QUANT, true>(p, row, c0, v, gamma, rstd);
  else store_run<CHANNELS, SKIP, QUANT, false>(p, row, c0, v, gamma, rstd);
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
        y[j] = (rstd == 0.0f ? v * 0.0f : v) * __bfloat162float(p.gamma[c]);  // (squares that overflow give zeros)
        if (p.residual != nullptr) p.residual[row * p.ld_residual + c] = __float2bfloat16_rn(v);
        if (p.out != nullptr) p.out[row * p.ld_out + c] = __float2bfloat16_rn(y[j] * rstd);
      }
      amax = max(amax, magnitude_bits(y[j]));
    }
    if (p.q != nullptr) {
      float scale, inverse;
      if (!fp8_norm_block_scale(__reduce_max_sync(0xFFFFFFFFu, amax), rstd, scale, inverse)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] *= rstd;
      }
      if (lane == 0) p.scale[block * p.ld_scale + row] = scale;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = block * kFp8Block + 32 * j + lane;
        if (c < p.width) p.q[row * p.ld_q + c] = static_cast<uint8_t>(fp8_pack2(y[j] * inverse, 0.0f));
      }
    }
  }
}

template <int GROUPS, int THREADS>
void launch_words(const RmsParams& p, cudaStream_t st) {
  const dim3 block(THREADS == 32 ? 32 * kWarpsPerBlock : 256);
  const dim3 grid(static_cast<unsigned>(ceil_div_ll(p.rows, block.x / THREADS)));
  const bool skip = p.skip != nullptr, quant = p.q != nullptr;
  if (skip && quant) launch_dependent(rms_norm_kernel<GROUPS, THREADS, true, true>, grid, block, 0, st, p);
  else if (skip) launch_dependent(rms_norm_kernel<GROUPS, THREADS, true, false>, grid, block, 0, st, p);
  else if (quant) launch_dependent(rms_norm_kernel<GROUPS, THREADS, false, true>, grid, block, 0, st, p);
  else launch_dependent(rms_norm_kernel<GROUPS, THREADS, false, false>, grid, block, 0, st, p);
}

template <int CHANNELS, bool MANY>
void launch_odd(const RmsParams& p, dim3 grid, dim3 block, cudaStream_t st) {
  const bool skip = p.skip != nullptr, quant = p.q != nullptr;
  if (skip && quant) launch_dependent(rms_norm_odd_kernel<CHANNELS, true, true, MANY>, grid, block, 0, st, p);
  else if (skip) launch_dependent(rms_norm_odd_kernel<CHANNELS, true, false, MANY>, grid, block, 0, st, p);
  else if (quant) launch_dependent(rms_norm_odd_kernel<CHANNELS, false, true, MANY>, grid, block, 0, st, p);
  else launch_dependent(rms_norm_odd_kernel<CHANNELS, false, false, MANY>, grid, block, 0, st, p);
}

template <int CHANNELS>
void launch_odd(const RmsParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.rows)), block(static_cast<unsigned>(32 * ceil_div_ll(p.width, 32 * CHANNELS)));
  launch_odd<CHANNELS, false>(p, grid, block, st);
}

// Rows of one or two warps, up to four warps a CTA as long as there are eight CTAs for every SM.
void launch_odd_narrow(const RmsParams& p, cudaStream_t st) {
  const unsigned warps = p.width <= 256 ? 1 : 2;
  unsigned rows_each = 1;
  while (2 * rows_each * warps <= 4 && p.rows / (2 * rows_each) >= 8LL * sm_count()) rows_each *= 2;
  const dim3 grid(static_cast<unsigned>(ceil_div_ll(p.rows, rows_each)));
  launch_odd<8, true>(p, grid, dim3(32 * warps, rows_each), st);
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
  const bool words = (width % 8) == 0 && rows_aligned16(in, ld_in) && rows_aligned16(skip, ld_skip) &&
                     rows_aligned16(out, ld_out) && rows_aligned16(residual, ld_residual) && aligned16(gamma) &&
                     (q_out == nullptr || ((reinterpret_cast<uintptr_t>(q_out) % 8) == 0 && (ld_q % 8) == 0));
  if (words && width <= 16384) {
    // One warp per row up to 2048 channels, but not where there are fewer rows than SMs: a CTA then shares the row out.
    if (width <= 2048 && (rows > sm_count() || width <= 256)) {
      if (width <= 128) launch_words<1, 16>(p, st);
      else if (width <= 256) launch_words<1, 32>(p, st);
      else if (width <= 512) launch_words<2, 32>(p, st);
      else if (width <= 1024) launch_words<4, 32>(p, st);
      else if (width <= 1536) launch_words<6, 32>(p, st);
      else launch_words<8, 32>(p, st);
    } else if (width <= 2048) {
      launch_words<1, 256>(p, st);
    } else if (width <= 4096) {
      launch_words<2, 256>(p, st);
    } else if (width <= 8192) {
      launch_words<4, 256>(p, st);
    } else {
      launch_words<8, 256>(p, st);
    }
    return launch_status();
  }
  if (width <= 512) {
    launch_odd_narrow(p, st);
    return launch_status();
  }
  if (width <= 8192) {
    launch_odd<8>(p, st);
    return launch_status();
  }
  if (width <= 16384) {
    launch_odd<16>(p, st);
    return launch_status();
  }
  launch_dependent(rms_norm_any_kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st, p);
  return launch_status();
}

}  // namespace lc0b200
