// Block-scaled e4m3 product on the tensor cores (sm_100a):
//   out[m,n] = act(bias[n] + sum_b sa[b,m] * sw[n/128,b] * P_b[m,n]),   P_b = the product over 128-block b of k.
// tcgen05.mma (kind::f8f6f4, f32 accumulation) forms one P_b at a time in tensor memory, overwriting; the epilogue warps
// read it back, scale it and keep the running sum in registers, so the f32 scales need no restriction and the sum over
// blocks is a plain fp32 chain in the order of b.  The scale of a block is ONE number per output row and 128 columns,
// and an epilogue thread owns one row: one fused multiply-add per element and block.
//
// gemm_fp8_kernel (many rows): persistent, tiles of 128 x BN per CTA, or 256 x 256 per CTA pair (cta_group::2; each CTA
// loads its own rows of A and its own half of W with plain TMA loads, none is multicast).  Warp 0 loads (one elected
// lane), warp 1 issues the MMAs, warps 2 and 3 bring the scales, warps 4 and up are the epilogue: two per TMEM lane quarter,
// each with half of the columns.  Bound by the way of a partial through the epilogue and back (710 cycles a block against
// 512 of MMA, with the two partials that fit), then by what ends a tile (3500 cycles, 8400 with mish), and back to back by
// the power limit.  Ten launches after a rest / launches back to back for seconds, us: 32768 x 1024 x 4096: 125 (2200 TFLOP/s) /
// 146; 65536 x 1024 x 1024: 74 / 87; 32768 x 1536 x 1024 with mish: 88 / 89; 32768 x 1024 x 1024: 42 / 45, to f32 70 / 71.
// Other figures of single kernels here are of the first kind.
// gemm_fp8_few_kernel (few rows): further down.  Bound by the weight's bytes, or by latency: 1 x 4096 x 4096 in 6.3 us,
// 1 x 16384 x 16384 in 48 (5.6 TB/s).
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "fp8.cuh"
#include "gemm_fp8.h"
#include "ptx.cuh"
#include "tensormap.h"

namespace lc0b200 {

namespace {

constexpr int kBM = 128;           // rows of a CTA's tile = TMEM lanes
constexpr int kRowBytes = 128;     // one swizzle row = one 128-block of k
constexpr int kMmaK = 32;          // k per tcgen05.mma
constexpr int kGroupBytes = 32 * kRowBytes;  // staging of 32 rows x 64 bf16 columns, or 32 x 32 f32

template <int CTAS>
__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  if (CTAS == 2) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Waits for this thread's tensor-memory loads; names the registers, so that no use of them can move above it.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// 32 lanes x 16 or 32 columns of tensor memory.
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&v)[32]) { ptx::tmem_ld_32x32(taddr, v); }

__device__ __forceinline__ uint64_t pack_f32x2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t both_f32x2(float x) { return pack_f32x2(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// acc += a * b, both halves.
__device__ __forceinline__ void fma_f32x2(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

// Arrival at a barrier of another CTA of the cluster that publishes no memory: it says that tensor-memory loads whose
// values are in registers are done.  Relaxed, because a release at cluster scope is a memory barrier that waits for
// everything this thread has in flight, once per k block.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// After a wait that ran out, each for a millisecond at the most:
constexpr uint64_t kDrainLimitNs = 1000000;
// The loads under way still write into this CTA's memory.  Waits for the last one of every stage; `stage` and `phase` are where
// the next load would have gone.  The loads of a pair complete on the leader's barriers, and its peer may have issued one
// that the leader did not get to: both rest for the whole millisecond.
template <int CTAS>
__device__ __forceinline__ void drain_loads(uint32_t bar_full, int stages, int stage, uint32_t phase) {
  const uint64_t start = ptx::globaltimer_ns();
  for (int s = 0; CTAS == 1 && s < stages; ++s) {
    const uint32_t parity = s < stage ? phase : phase ^ 1u;
    while (!ptx::mbar_try_wait(bar_full + 8 * s, parity) && ptx::globaltimer_ns() - start < kDrainLimitNs) {
    }
  }
  while (CTAS == 2 && ptx::globaltimer_ns() - start < kDrainLimitNs) {
  }
}
// The MMAs under way still read shared memory and write tensor memory (a pair's in both CTAs).  Called by the lane that issued
// them: its commit arrives at `bar_done` once they have ended.
template <int CTAS>
__device__ __forceinline__ void drain_mmas(uint32_t bar_done) {
  if (CTAS == 2) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(ptx::map_to_cta(bar_done, 0u)) : "memory");
  } else {
    ptx::tc_commit<1>(bar_done);
  }
  const uint64_t start = ptx::globaltimer_ns();
  while (!ptx::mbar_try_wait(bar_done, 0u) && ptx::globaltimer_ns() - start < kDrainLimitNs) {
  }
}

template <int BN, int CTAS>
struct Tile {
  static_assert(CTAS == 1 || (CTAS == 2 && BN == 256), "CTA pairs share 256 x 256 tiles");
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBRows = BN / CTAS;
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // Block products in flight in tensor memory.  (A 256-wide tile as two half products with barriers of their own, so that
  // one is handed on while the other is multiplied, was measured slower: 163 us against 139 at 32768 x 1024 x 4096.
  // MMAs 128 wide are limited by their operand reads from shared memory.)
  static constexpr int kPartials = 512 / BN;
  static constexpr int kTmemCols = kPartials * BN;
  static constexpr int kEpilogueWarps = 8;
  static constexpr int kCols = BN / (kEpilogueWarps / 4);  // columns per epilogue thread: 128 or 64
  // Four warps in front of the epilogue: loads, MMAs, and two that fetch the scales.
  static constexpr int kThreads = 128 + 32 * kEpilogueWarps;
  // 128 running sums a thread do not fit into an even share of the registers (65536 / 384 threads = 168): the first
  // warpgroup gives some of its own up.  The shares add up to what the block was launched with.
  static constexpr bool kSplitRegs = kCols == 128;
  static constexpr int kLaunchRegs = 168, kFrontRegs = 40, kEpilogueRegs = 232;
  static_assert(128 * kFrontRegs + 256 * kEpilogueRegs <= 384 * kLaunchRegs, "the register shares exceed the launch's");
  static constexpr int kGroups = kCols / 64;
  static constexpr int kStagingBytes = kEpilogueWarps * kGroups * kGroupBytes;
  static constexpr int kBarrierBytes = 512;
  static constexpr int kScaleCols = (BN + kFp8Block - 1) / kFp8Block;
  static constexpr int kScaleBytes = kScaleCols * kBM * 4;         // one product of two scales per row and 128 columns
  static constexpr int kFixedBytes = kStagingBytes + kBarrierBytes + kPartials * kScaleBytes;
  static constexpr int kFit = (227 * 1024 - kFixedBytes) / kStageBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static_assert(kStages >= 3, "pipeline too shallow");
  static constexpr int kSmemBytes = kStages * kStageBytes + kFixedBytes;
};

struct FpParams {
  GemmFp8 g;
  int tma_store;  // bf16 result with a base, pitch and width that a tensor map can store
  unsigned int* status;
  const bf16* a_bf16;  // few-row kernel on bf16 rows: they are quantised on the way in (g.a, g.a_scale are not read)
  long long ld_a_bf16;
};

// Columns that the MMAs of the tile at tile_n0 cover: a ragged last tile costs its own width rounded up to 32.
template <int BN>
__device__ __forceinline__ int mma_width(int n, int tile_n0) {
  const int left = n - tile_n0;
  return left >= BN ? BN : ((left + 31) & ~31);
}

// mish(x) = x n / (n + 2), n = e^x (e^x + 2) (formula: bt4/kernels/layer_norm.py:61-69), of PAIRS packed pairs in step: each
// phase is a run of independent operations.  One reciprocal serves four values (1 / a = b c d / (a b c d)).  The exponential
// is taken of min(x, 10): there n / (n + 2) rounds to 1, and the product of four denominators stays below 6e34, so that its
// reciprocal is far from the values that the fast reciprocal flushes to zero.
template <int PAIRS>
__device__ __forceinline__ void mish_pairs(uint64_t* x) {
  const uint64_t two = both_f32x2(2.0f), log2e = both_f32x2(1.4426950408889634f);
  uint64_t n[PAIRS], d[PAIRS], r[PAIRS / 2];
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    float lo, hi;
    unpack_f32x2(mul_f32x2(x[j], log2e), lo, hi);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(lo) : "f"(fminf(lo, 14.42695f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(fminf(hi, 14.42695f)));
    n[j] = pack_f32x2(__float_as_uint(lo), __float_as_uint(hi));
  }
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) n[j] = mul_f32x2(n[j], add_f32x2(n[j], two));
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) d[j] = add_f32x2(n[j], two);
#pragma unroll
  for (int j = 0; j < PAIRS; j += 2) {
    float lo, hi, inverse;
    unpack_f32x2(mul_f32x2(d[j], d[j + 1]), lo, hi);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(lo * hi));
    r[j / 2] = pack_f32x2(__float_as_uint(inverse * hi), __float_as_uint(inverse * lo));
  }
#pragma unroll
  for (int j = 0; j < PAIRS; j += 2) {  // n / (n + 2) first: x n may overflow
    x[j] = mul_f32x2(x[j], mul_f32x2(n[j], mul_f32x2(r[j / 2], d[j + 1])));
    x[j + 1] = mul_f32x2(x[j + 1], mul_f32x2(n[j + 1], mul_f32x2(r[j / 2], d[j])));
  }
}

// Bias and activation of 32 columns from col0 on, as packed pairs; columns past the matrix edge get no bias (they are not
// stored).  ACT is fixed at compile time: what a tile executes once has to be fetched once, and jumping over the other
// activations cost 300 cycles for 32 columns that had nothing to do.
template <int ACT>
__device__ __forceinline__ void finish32(uint64_t (&y)[16], const GemmFp8& g, int col0) {
  if (g.bias != nullptr) {
    if (col0 + 32 <= g.n && aligned16_dev(g.bias)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(g.bias + col0) + i);
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * i + j] = add_f32x2(y[4 * i + j], pack_f32x2(words[j] << 16, words[j] & 0xFFFF0000u));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = col0 + 2 * j;
        y[j] = add_f32x2(y[j], pack_f32x2(__float_as_uint(c < g.n ? __bfloat162float(g.bias[c]) : 0.0f),
                                          __float_as_uint(c + 1 < g.n ? __bfloat162float(g.bias[c + 1]) : 0.0f)));
      }
    }
  }
  if (ACT == LC0B200_ACT_MISH) {
    mish_pairs<8>(y);
    mish_pairs<8>(y + 8);
  } else if (ACT != LC0B200_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float lo, hi;
      unpack_f32x2(y[j], lo, hi);
      if (ACT == LC0B200_ACT_RELU) {  // NaN stays
        lo = lo < 0.0f ? 0.0f : lo;
        hi = hi < 0.0f ? 0.0f : hi;
      } else {
        lo = act_swish(lo);
        hi = act_swish(hi);
      }
      y[j] = pack_f32x2(__float_as_uint(lo), __float_as_uint(hi));
    }
  }
}

__device__ __forceinline__ uint32_t pack_bf16x2(uint64_t pair) {
  float lo, hi;
  unpack_f32x2(pair, lo, hi);
  return lc0b200::pack_bf16x2(lo, hi);
}

// The tiles of a CTA (pair), every num_groups-th: row and column of the tile without a division each.
struct TileWalk {
  long long tile, m;
  int n;
  __device__ TileWalk(long long first, int n_tiles) : tile(first), m(first / n_tiles), n(static_cast<int>(first % n_tiles)) {}
  __device__ void next(uint32_t groups, int step_m, int step_n, int n_tiles) {
    tile += groups;
    m += step_m;
    n += step_n;
    if (n >= n_tiles) {
      n -= n_tiles;
      ++m;
    }
  }
};

template <int BN, int CTAS, int ACT>
__global__ void __launch_bounds__(Tile<BN, CTAS>::kThreads, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_out, const FpParams p) {
  using T = Tile<BN, CTAS>;
  constexpr int kStages = T::kStages;
  constexpr int kPartials = T::kPartials;
  constexpr int kTileM = kBM * CTAS;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = ptx::smem_u32(smem_raw);
  const uint32_t smem_a = smem_base;
  const uint32_t smem_b = smem_base + kStages * T::kABytes;
  const uint32_t staging_base = smem_base + kStages * T::kStageBytes;
  const uint32_t bar_base = staging_base + T::kStagingBytes;
  const uint32_t bar_full = bar_base;                                   // [kStages] (leader CTA's are used)
  const uint32_t bar_empty = bar_base + 8 * kStages;                    // [kStages]
  const uint32_t bar_part_full = bar_base + 16 * kStages;               // [kPartials] product and scales are there
  const uint32_t bar_part_empty = bar_part_full + 8 * kPartials;        // [kPartials] (leader CTA's are used)
  const uint32_t bar_scale_empty = bar_part_empty + 8 * kPartials;      // [kPartials]
  const uint32_t tmem_slot = bar_scale_empty + 8 * kPartials;
  const uint32_t scale_base = bar_base + T::kBarrierBytes;              // [kPartials][kScaleCols][kBM] f32
  const uint32_t bar_done = tmem_slot + 8;  // for drain_mmas alone
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_raw + (tmem_slot + 4 - smem_base));
  static_assert(16 * kStages + 24 * kPartials + 16 <= T::kBarrierBytes, "barrier area too small");
  grid_dependency_release();
  if ((smem_base & 1023u) != 0u) {  // never seen; refuse loudly rather than mis-swizzle
    if (threadIdx.x == 0 && atomicCAS(&p.status[0], 0u, kDeviceSmemMisaligned) == 0u) p.status[1] = smem_base;
    return;
  }

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = (CTAS == 2) ? ptx::cluster_ctarank() : 0u;  // rank 0 leads: issues the MMAs, owns the barriers
  const uint32_t group = blockIdx.x / CTAS;
  const uint32_t num_groups = gridDim.x / CTAS;
  const GemmFp8& g = p.g;
  const int n_tiles = (g.n + BN - 1) / BN;
  const long long num_tiles = ceil_div_ll(g.m, kTileM) * n_tiles;
  const int k_blocks = (g.k + kFp8Block - 1) / kFp8Block;
  const int step_m = static_cast<int>(num_groups) / n_tiles, step_n = static_cast<int>(num_groups) % n_tiles;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < kPartials; ++a) {
      ptx::mbar_init(bar_part_full + 8 * a, 2);  // the MMAs' completion and a scale warp
      ptx::mbar_init(bar_part_empty + 8 * a, T::kEpilogueWarps * CTAS);
      ptx::mbar_init(bar_scale_empty + 8 * a, T::kEpilogueWarps);
    }
    ptx::mbar_init(bar_done, 1);
    ptx::mbar_init_fence();
    ptx::prefetch_tensormap(&map_a);
    ptx::prefetch_tensormap(&map_w);
    if (p.tma_store) ptx::prefetch_tensormap(&map_out);
  }
  if (warp == 1) {
    if (CTAS == 2) {
      ptx::tmem_alloc_pair(tmem_slot, T::kTmemCols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, T::kTmemCols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (CTAS == 2) ptx::cluster_sync();  // the peer's barriers exist before anything signals them
  ptx::tc_fence_after_sync();
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  grid_dependency_wait();

  if (warp < 4) {
    if (T::kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kFrontRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ loads: the warp follows the loop, one lane issues
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long tile = group; tile < num_tiles && ok; tile += num_groups) {
        const int m0 = static_cast<int>(tile / n_tiles) * kTileM + static_cast<int>(rank) * kBM;
        const int tile_n0 = static_cast<int>(tile % n_tiles) * BN;
        // A pair splits the weight tile's rows between its CTAs.
        const int n0 = tile_n0 + static_cast<int>(rank) * (mma_width<BN>(g.n, tile_n0) / CTAS);
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = ptx::mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status, 0x1100u + stage);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          if (ptx::elect_one()) {
            const uint32_t full = (CTAS == 2) ? ptx::map_to_cta(bar_full + 8 * stage, 0u) : bar_full + 8 * stage;
            if (rank == 0) ptx::mbar_expect_tx(bar_full + 8 * stage, T::kStageBytes * CTAS);
            ptx::tma_load_2d<CTAS>(smem_a + stage * T::kABytes, &map_a, kb * kFp8Block, m0, full);
            ptx::tma_load_2d<CTAS>(smem_b + stage * T::kBBytes, &map_w, kb * kFp8Block, n0, full);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) drain_loads<CTAS>(bar_full, kStages, stage, phase);
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMAs (leader CTA only): one partial per k block
      // One lane runs the whole loop: it may give up by itself.  (With the warp in step around an elected lane every wait has to
      // be followed by a vote: 2048 x 1024 x 4096 on 128-wide tiles in 15.6 us, 14.3 without votes, 13.1 so; on pair tiles
      // the three are within half a per cent.)
      if (rank == 0 && ptx::elect_one()) {
        int stage = 0, part = 0;
        uint32_t phase = 0, part_phase = 0;
        bool ok = true;
        for (long long tile = group; tile < num_tiles && ok; tile += num_groups) {
          const int tile_n0 = static_cast<int>(tile % n_tiles) * BN;
          const uint32_t idesc = ptx::instr_desc(1u, 0u, 0u, static_cast<uint32_t>(kTileM),
                                                 static_cast<uint32_t>(mma_width<BN>(g.n, tile_n0)));
          for (int kb = 0; kb < k_blocks; ++kb) {
            // The operands first: they are there early, and the look at their barrier is off the path from a freed partial.
            ok = ptx::mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, 0x1300u + stage);
            const uint64_t a_desc = ptx::smem_desc_sw128(smem_a + stage * T::kABytes, 16, 1024);
            const uint64_t b_desc = ptx::smem_desc_sw128(smem_b + stage * T::kBBytes, 16, 1024);
            ok = ok && ptx::mbar_wait(bar_part_empty + 8 * part, part_phase ^ 1u, abort_flag, p.status, 0x1200u + part);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int j = 0; j < kFp8Block / kMmaK; ++j) {
              mma_e4m3<CTAS>(tmem_base + part * BN, a_desc + j * (kMmaK >> 4), b_desc + j * (kMmaK >> 4), idesc, j > 0 ? 1u : 0u);
            }
            ptx::tc_commit<CTAS>(bar_part_full + 8 * part);
            ptx::tc_commit<CTAS>(bar_empty + 8 * stage);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
            if (++part == kPartials) {
              part = 0;
              part_phase ^= 1u;
            }
          }
        }
        if (!ok) drain_mmas<CTAS>(bar_done);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------ scales: a_scale[row] * w_scale of each k block
      // Two warps take the k blocks in turn; the scales of a block wait in shared memory beside its partial, behind the
      // same barrier.  (Epilogue warps that fetched their own were slower, 176 us against 137 at 32768 x 1024 x 4096 in the
      // worst schedule: a wait for tensor memory may then also wait for a global load.)
      const int first = warp - 2;
      int part = first;
      uint32_t phase = 0;
      TileWalk walk(group, n_tiles);
      int kb = first;
      while (true) {
        while (kb >= k_blocks) {
          kb -= k_blocks;
          walk.next(num_groups, step_m, step_n, n_tiles);
        }
        if (walk.tile >= num_tiles) break;
        const long long row0 = walk.m * kTileM + rank * kBM + lane;
        const int column = walk.n * BN;
        float a[4], w[T::kScaleCols];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = row0 + 32 * i < g.m ? __ldg(g.a_scale + kb * g.ld_a_scale + row0 + 32 * i) : 0.0f;
#pragma unroll
        for (int h = 0; h < T::kScaleCols; ++h) {
          const int n0 = column + h * kFp8Block;
          w[h] = n0 < g.n ? __ldg(g.w_scale + (n0 / kFp8Block) * g.ld_w_scale + kb) : 0.0f;
        }
        bool ok = ptx::mbar_wait(bar_scale_empty + 8 * part, phase ^ 1u, abort_flag, p.status, 0x1500u + part);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < T::kScaleCols; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = scale_base + part * T::kScaleBytes + (h * kBM + 32 * i + lane) * 4;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(a[i] * w[h]) : "memory");
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_part_full + 8 * part);
        part += 2;
        if (part >= kPartials) {
          part = first;
          phase ^= 1u;
        }
        kb += 2;
      }
      __syncwarp();
    }
  } else {
    if (T::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kEpilogueRegs));
    // ------------------------------------------------------------ epilogue: scale and sum the partials, then store
    const int ew = warp - 4;
    const int quarter = warp & 3;  // TMEM lane quarter this warp may read
    const int half = ew >> 2;
    const uint32_t staging = staging_base + ew * T::kGroups * kGroupBytes;
    const uint32_t tmem_row = tmem_base + half * T::kCols + (static_cast<uint32_t>(quarter * 32) << 16);
    int part = 0;
    uint32_t part_phase = 0;
    bool ok = true;
    const uint32_t my_scale = scale_base + ((half * T::kCols / kFp8Block) * kBM + quarter * 32 + lane) * 4;
    // Running sums as packed pairs of fp32: one packed multiply-add for two columns.
    constexpr int kChunks = T::kCols / 32;
    static_assert(kChunks % 2 == 0, "a block's first columns go to the first buffer");
    uint64_t acc[T::kCols / 2];
    float scale = 0.0f;
    // Waits for the next partial and fetches its scale.  A wait that ran out changes nothing yet: lanes must not part before
    // the tensor-memory loads that follow (of whatever is there), and the vote on `ok` comes after them, where it costs nothing.
    auto begin_block = [&](float& block_scale) {
      ok = ptx::mbar_wait(bar_part_full + 8 * part, part_phase, abort_flag, p.status, 0x1400u + part);
      ptx::tc_fence_after_sync();
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(block_scale) : "r"(my_scale + part * T::kScaleBytes) : "memory");
    };
    // Hands a partial that has been read back to the MMAs, its scales back to their warps.
    auto end_block = [&](int which) {
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) mbar_arrive_cluster_relaxed(ptx::map_to_cta(bar_part_empty + 8 * which, 0u));
        else ptx::mbar_arrive(bar_part_empty + 8 * which);
        ptx::mbar_arrive(bar_scale_empty + 8 * which);
      }
    };
    auto take_part = [&]() {
      const int taken = part;
      if (++part == kPartials) {
        part = 0;
        part_phase ^= 1u;
      }
      return taken;
    };
    constexpr int kTaken = CTAS == 2 ? 1 : 0;  // blocks of a tile in front of the loop; tiles of one CTA are about one to a CTA
    long long row = 0;  // of the tile whose sums are being formed or finished
    int n0 = 0;
    // Stores the 32 columns from col0 on, chunk c of the tile, or leaves them in the staging buffers of a tensor map's store.
    auto store_chunk = [&](int c, int col0, uint64_t (&y)[16]) {
      if (p.tma_store) {
        // Row `lane` of the group's 32 x 128-byte buffer, 16-byte chunk i at i ^ (lane & 7): the 128-byte swizzle.
        const uint32_t row_addr = staging + (c >> 1) * kGroupBytes + lane * kRowBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ptx::st_shared_v4(row_addr + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4), pack_bf16x2(y[4 * i]),
                            pack_bf16x2(y[4 * i + 1]), pack_bf16x2(y[4 * i + 2]), pack_bf16x2(y[4 * i + 3]));
        }
        return;
      }
      // f32 results and rows a tensor map cannot address: turn the 32 x 32 block in shared memory (element c of
      // row r at c ^ r, no bank conflicts either way) and write whole rows, 32 neighbouring elements a store, eight rows in
      // flight (20000 x 1858 x 1024 with mish, back to back: 93 us, a quarter more row by row).
      float* block = reinterpret_cast<float*>(smem_raw + (staging - smem_base));
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float lo, hi;
        unpack_f32x2(y[j], lo, hi);
        block[lane * 32 + ((2 * j) ^ lane)] = lo;
        block[lane * 32 + ((2 * j + 1) ^ lane)] = hi;
      }
      __syncwarp();
      const int rows = static_cast<int>(min(static_cast<long long>(32), g.m - (row - lane)));
      if (col0 + lane < g.n) {
        const long long at = (row - lane) * g.ldc + col0 + lane;
        if (g.out_kind == LC0B200_OUT_F32) {
          float* dst = reinterpret_cast<float*>(g.out) + at;
#pragma unroll 8
          for (int r = 0; r < rows; ++r) dst[r * g.ldc] = block[r * 32 + (lane ^ r)];
        } else {
          bf16* dst = reinterpret_cast<bf16*>(g.out) + at;
#pragma unroll 8
          for (int r = 0; r < rows; ++r) dst[r * g.ldc] = __float2bfloat16_rn(block[r * 32 + (lane ^ r)]);
        }
      }
      __syncwarp();
    };

    // A tile's first block sets the sums, where a tile ends behind another's: no additions to zeros.  (Started from zeros as
    // tiles of one CTA are, 262144 x 1536 x 1024 takes 535 us back to back instead of 515.)
    auto take_first = [&]() {
      begin_block(scale);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) return;
      const int this_part = take_part();
      const uint64_t scale2 = both_f32x2(scale);
      uint32_t w[32];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        ptx::tmem_ld_32x32(tmem_row + this_part * BN + 32 * c, w);
        tmem_wait(w);
        if (c + 1 == kChunks) end_block(this_part);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[c * 16 + j] = mul_f32x2(pack_f32x2(w[2 * j], w[2 * j + 1]), scale2);
      }
    };
    // After a tile's last block: bias, activation and store, 32 columns at a time.  (With the next tile's first block taken into
    // the registers that this frees, 32 columns at a time as well, 262144 x 1536 x 1024 gained half a per cent without an
    // activation and lost 3 with mish, and results that no tensor map stores lost 4 to 10 to the larger kernel.)
    auto finish = [&]() {
      if (p.tma_store) {
        if (lane == 0) ptx::bulk_wait_read<0>();  // the staging buffers are free once the last tile's stores have read them
        __syncwarp();
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int col0 = n0 + 32 * c;
        if (col0 >= g.n) break;
        uint64_t y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = acc[c * 16 + j];
        finish32<ACT>(y, g, col0);
        store_chunk(c, col0, y);
      }
      if (p.tma_store) {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < T::kGroups; ++i) {
            if (n0 + 64 * i < g.n) ptx::tma_store_2d(&map_out, staging + i * kGroupBytes, n0 + 64 * i, static_cast<int>(row));
          }
          ptx::bulk_commit();
        }
      }
    };

    TileWalk walk(group, n_tiles);
    while (walk.tile < num_tiles && ok) {
      if (kTaken > 0) take_first();
      if (!ok) break;
      row = walk.m * kTileM + rank * kBM + quarter * 32 + lane;
      n0 = walk.n * BN + half * T::kCols;
      // 32 columns at a time: while they are added, the next 32 are on their way, across the k blocks too (a partial is
      // handed back, and the next one's first columns asked for, before the last additions).  Columns past the matrix
      // edge hold anything and are not stored.
      if (kTaken == 0) {
#pragma unroll
        for (int i = 0; i < T::kCols / 2; ++i) acc[i] = 0ull;
      }
      uint32_t v[2][32];
      if (k_blocks > kTaken) {
        begin_block(scale);
        ptx::tmem_ld_32x32(tmem_row + part * BN, v[0]);
        ok = __all_sync(0xFFFFFFFFu, ok);
      }
      for (int kb = kTaken; kb < k_blocks && ok; ++kb) {
        const uint64_t scale2 = both_f32x2(scale);
        const int this_part = take_part();
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          tmem_wait(v[c & 1]);
          if (c + 1 < kChunks) {
            ptx::tmem_ld_32x32(tmem_row + this_part * BN + 32 * (c + 1), v[(c + 1) & 1]);
          } else {
            end_block(this_part);
            if (kb + 1 < k_blocks) {
              begin_block(scale);
              ptx::tmem_ld_32x32(tmem_row + part * BN, v[0]);
              ok = __all_sync(0xFFFFFFFFu, ok);
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) fma_f32x2(acc[c * 16 + j], pack_f32x2(v[c & 1][2 * j], v[c & 1][2 * j + 1]), scale2);
        }
      }
      if (!ok) {
        tmem_wait(v[0]);  // asked for all the same, and not to arrive in registers that hold something else
        break;
      }
      walk.next(num_groups, step_m, step_n, n_tiles);
      if (n0 < g.n) finish();
    }
    if (p.tma_store && lane == 0) ptx::bulk_wait_read<0>();  // staging must outlive the last store's read
    __syncwarp();
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (CTAS == 2) ptx::cluster_sync();  // neither CTA leaves while the other can signal its barriers or read its memory
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    if (CTAS == 2) ptx::tmem_dealloc_pair(tmem_base, T::kTmemCols);
    else ptx::tmem_dealloc(tmem_base, T::kTmemCols);
  }
}

// ---------------------------------------------------------------- few rows
//
// Too few rows of A for 128-row tiles to fill the SMs: the weight's bytes are the work, and a 128-row tile of A would be
// mostly padding.  So the roles are turned round: 128 weight rows are the M side of the MMA, NT = 16, 32 or 64 tokens its
// N side, and out^T comes out: an epilogue thread owns one weight row, a block's scales are one product per token.  The k
// blocks of a tile are split over the CTAs of a cluster, so that a layer of a few tiles still pulls on the memory of every
// SM.  Tokens 4 i .. 4 i + 3 are finished by CTA i mod S: each CTA writes its sums for them straight into that CTA's
// shared memory, one cluster barrier later the owner adds the S pieces in the order of the CTAs (the same bits every time).
// (Fetching the pieces from the other CTAs instead took 2600 cycles a token and a second barrier of 2000.)  A CTA takes half
// of an SM's shared memory and registers: two are resident, one loads while the other finishes.
constexpr int kMaxSplits = 8;  // CTAs of a cluster (the portable limit)

template <int NT>
struct Few {
  static constexpr int kWBytes = kBM * kRowBytes;
  static constexpr int kStageBytes = kWBytes + NT * kRowBytes;
  static constexpr int kPartials = 4;
  static constexpr int kTmemCols = kPartials * NT;  // 64, 128, 256
  // Epilogue warps: four, or eight with half of the columns each.
  static constexpr int kEpilogueWarps = NT == 64 ? 8 : 4;
  static constexpr int kCols = NT / (kEpilogueWarps / 4);  // 16 or 32
  static constexpr int kThreads = 128 + 32 * kEpilogueWarps;  // in front: loads, MMAs, two for scales
  static constexpr int kBarrierBytes = 512;
  static constexpr int kScaleBytes = NT * 4;
  // What the CTAs of a cluster write here: [CTA][own groups of four tokens][weight row][4] f32.  A CTA owns one group at the
  // least, also where there are more CTAs than groups.
  static constexpr int kSumBytes = (NT / 4 > kMaxSplits ? NT / 4 : kMaxSplits) * kBM * 16;
  static constexpr int kFixedBytes = kSumBytes + kBarrierBytes + kPartials * kScaleBytes;
  static constexpr int kStages = (113 * 1024 - kFixedBytes) / kStageBytes;
  static_assert(kStages >= 3 && kStages <= 8, "pipeline depth");
  static constexpr int kSmemBytes = kStages * kStageBytes + kFixedBytes;
};

__device__ __forceinline__ float finish_one(float y, const GemmFp8& g, int column) {
  if (g.bias != nullptr) y += __bfloat162float(g.bias[column]);
  return fp8_activate(y, g.activation);
}

__device__ __forceinline__ void store_one(float y, const GemmFp8& g, long long at) {
  if (g.out_kind == LC0B200_OUT_F32) reinterpret_cast<float*>(g.out)[at] = y;
  else reinterpret_cast<bf16*>(g.out)[at] = __float2bfloat16_rn(y);
}

// BF16_A: the dense layer on bf16 rows in one launch.  The scale warps bring the tokens' rows of a k block, apply the
// block rule of quantize_fp8 (the same bits) and write the codes where the tensor map would have put them.  Every weight
// tile does this again for its tokens, from the L2: worth it for the few tokens of one MMA column group (two launches
// for 8 tokens, 8192 x 2048: 9.2 us on the GPU and 12.6 us a call).
template <int NT, bool BF16_A>
__global__ void __launch_bounds__(Few<NT>::kThreads, 2)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const FpParams p) {
  using T = Few<NT>;
  constexpr int kStages = T::kStages;
  constexpr int kPartials = T::kPartials;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = ptx::smem_u32(smem_raw);
  const uint32_t smem_w = smem_base;
  const uint32_t smem_a = smem_base + kStages * T::kWBytes;
  const uint32_t sums = smem_base + kStages * T::kStageBytes;
  const uint32_t bar_base = sums + T::kSumBytes;
  const uint32_t bar_full = bar_base;                               // [kStages]
  const uint32_t bar_empty = bar_base + 8 * kStages;                // [kStages]
  const uint32_t bar_part_full = bar_base + 16 * kStages;           // [kPartials] product and scales are there
  const uint32_t bar_part_empty = bar_part_full + 8 * kPartials;    // [kPartials]
  const uint32_t tmem_slot = bar_part_empty + 8 * kPartials;
  const uint32_t scale_base = bar_base + T::kBarrierBytes;          // [kPartials][NT] f32
  const uint32_t bar_done = tmem_slot + 8;  // for drain_mmas alone
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_raw + (tmem_slot + 4 - smem_base));
  static_assert(16 * kStages + 16 * kPartials + 16 <= T::kBarrierBytes, "barrier area too small");
  grid_dependency_release();

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int split_bits = 31 - __clz(static_cast<int>(ptx::cluster_nctaid()));  // S is a power of two
  const int splits = 1 << split_bits;
  const GemmFp8& g = p.g;
  // Token tiles of one weight tile are neighbours: they share its bytes in the L2.
  const int token_tiles = static_cast<int>((g.m + NT - 1) / NT);
  const int tile = static_cast<int>(blockIdx.x) / splits;
  const int n0 = tile / token_tiles * kBM;
  const long long m0 = static_cast<long long>(tile % token_tiles) * NT;
  const int tokens = static_cast<int>(min(static_cast<long long>(NT), g.m - m0));
  const int k_blocks = (g.k + kFp8Block - 1) / kFp8Block;
  const int kb_begin = static_cast<int>(static_cast<long long>(k_blocks) * rank / splits);
  const int kb_end = static_cast<int>(static_cast<long long>(k_blocks) * (rank + 1) / splits);
  const bool aligned = (smem_base & 1023u) == 0u;  // never false; then nothing is computed rather than mis-swizzled
  if (!aligned && threadIdx.x == 0 && atomicCAS(&p.status[0], 0u, kDeviceSmemMisaligned) == 0u) p.status[1] = smem_base;

  if (threadIdx.x == 0) {
    *abort_flag = aligned ? 0 : 1;
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, BF16_A ? 2 : 1);  // the copies, and the warp that writes the codes
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < kPartials; ++a) {
      ptx::mbar_init(bar_part_full + 8 * a, 2);   // the MMAs' completion and a scale warp
      ptx::mbar_init(bar_part_empty + 8 * a, T::kEpilogueWarps);
    }
    ptx::mbar_init(bar_done, 1);
    ptx::mbar_init_fence();
    ptx::prefetch_tensormap(&map_w);
    if (!BF16_A) ptx::prefetch_tensormap(&map_a);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, T::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_arrive_relaxed();  // "this CTA runs": awaited before the first write into another CTA's memory
  ptx::tc_fence_after_sync();
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  grid_dependency_wait();

  bool ok = aligned;
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb_begin; kb < kb_end && ok; ++kb) {
      ok = ptx::mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status, 0x2100u + stage);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      if (ptx::elect_one()) {
        ptx::mbar_expect_tx(bar_full + 8 * stage, BF16_A ? T::kWBytes : T::kStageBytes);
        ptx::tma_load_2d<1>(smem_w + stage * T::kWBytes, &map_w, kb * kFp8Block, n0, bar_full + 8 * stage);
        if (!BF16_A) {
          ptx::tma_load_2d<1>(smem_a + stage * NT * kRowBytes, &map_a, kb * kFp8Block, static_cast<int>(m0), bar_full + 8 * stage);
        }
      }
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok) drain_loads<1>(bar_full, kStages, stage, phase);
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = ptx::instr_desc(1u, 0u, 0u, kBM, NT);
    int stage = 0, part = 0;
    uint32_t phase = 0, part_phase = 0;
    for (int kb = kb_begin; kb < kb_end && ok; ++kb) {
      ok = ptx::mbar_wait(bar_part_empty + 8 * part, part_phase ^ 1u, abort_flag, p.status, 0x2200u + part);
      ok = ok && ptx::mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, 0x2300u + stage);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      if (ptx::elect_one()) {
#pragma unroll
        for (int j = 0; j < kFp8Block / kMmaK; ++j) {
          mma_e4m3<1>(tmem_base + part * NT, ptx::smem_desc_sw128(smem_w + stage * T::kWBytes + j * kMmaK, 16, 1024),
                      ptx::smem_desc_sw128(smem_a + stage * NT * kRowBytes + j * kMmaK, 16, 1024), idesc, j > 0 ? 1u : 0u);
        }
        ptx::tc_commit<1>(bar_empty + 8 * stage);
        ptx::tc_commit<1>(bar_part_full + 8 * part);
      }
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++part == kPartials) {
        part = 0;
        part_phase ^= 1u;
      }
    }
    if (!ok && ptx::elect_one()) drain_mmas<1>(bar_done);
    __syncwarp();
  } else if (warp < 4) {
    // Scales: two warps take the k blocks in turn; lane j holds the products of tokens j and j + 32.
    const float* w_scale = g.w_scale + (n0 / kFp8Block) * g.ld_w_scale;
    const int first = warp - 2;
    int part = first;
    uint32_t phase = 0;
    for (int kb = kb_begin + first; kb < kb_end && ok; kb += 2) {
      const float w = __ldg(w_scale + kb);
      if constexpr (BF16_A) {
        // A half-warp holds a token's block in step i: tokens 2 i and 2 i + 1.
        constexpr int kSteps = NT / 2;
        static_assert(kSteps % 4 == 0, "scales are worked out four steps at a time");
        const int lane16 = lane & 15, side = lane >> 4;
        const int channel = kb * kFp8Block + lane16 * 8;
        uint4 raw[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const bool here = 2 * i + side < tokens && channel < g.k;
          raw[i] = here ? __ldg(reinterpret_cast<const uint4*>(p.a_bf16 + (m0 + 2 * i + side) * p.ld_a_bf16 + channel)) : make_uint4(0u, 0u, 0u, 0u);
        }
        const int at = kb - kb_begin, stage = at % kStages;
        ok = ptx::mbar_wait(bar_part_empty + 8 * part, phase ^ 1u, abort_flag, p.status, 0x2500u + part) &&
             ptx::mbar_wait(bar_empty + 8 * stage, ((at / kStages) & 1u) ^ 1u, abort_flag, p.status, 0x2600u + stage);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
#pragma unroll
        for (int i0 = 0; i0 < kSteps; i0 += 4) {
          uint32_t m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) m[i] = magnitude_of_packed(packed_magnitude(raw[i0 + i]));
          float scale, inverse;
          fp8_block_scale(max_of_four_blocks(m), scale, inverse);
          if ((lane & 3) == 0) {
            const int token = 2 * (i0 + (lane16 >> 2)) + side;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(scale_base + part * T::kScaleBytes + token * 4), "f"(scale * w) : "memory");
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // Row `token` of the stage's 128-byte swizzled tile: 16-byte chunk c lies at c ^ (token & 7).
            const int token = 2 * (i0 + i) + side;
            const uint2 codes = codes8(raw[i0 + i], from_block(inverse, i));
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(smem_a + stage * NT * kRowBytes + token * kRowBytes +
                                                                (((lane16 >> 1) ^ (token & 7)) << 4) + (lane16 & 1) * 8),
                         "r"(codes.x), "r"(codes.y)
                         : "memory");
          }
        }
        ptx::fence_proxy_async_smem();  // the MMAs read the codes through the asynchronous proxy
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(bar_full + 8 * stage);
          ptx::mbar_arrive(bar_part_full + 8 * part);
        }
      } else {
        const float* a_scale = g.a_scale + kb * g.ld_a_scale + m0;
        const float a0 = lane < tokens ? __ldg(a_scale + lane) : 0.0f;
        const float a1 = NT > 32 && lane + 32 < tokens ? __ldg(a_scale + lane + 32) : 0.0f;
        ok = ptx::mbar_wait(bar_part_empty + 8 * part, phase ^ 1u, abort_flag, p.status, 0x2500u + part);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        const uint32_t dst = scale_base + part * T::kScaleBytes + lane * 4;
        if (lane < NT) asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst), "f"(a0 * w) : "memory");
        if (NT > 32) asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + 128), "f"(a1 * w) : "memory");
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_part_full + 8 * part);
      }
      part += 2;
      if (part >= kPartials) {
        part = first;
        phase ^= 1u;
      }
    }
    __syncwarp();
  }
  const int quarter = warp & 3;
  const int row = quarter * 32 + lane;  // of the weight tile
  const int col = NT == 64 ? ((warp - 4) >> 2) * T::kCols : 0;  // this warp's first token
  uint64_t acc[T::kCols / 2];  // running sums of two neighbouring tokens each
  if (warp >= 4) {
#pragma unroll
    for (int j = 0; j < T::kCols / 2; ++j) acc[j] = 0ull;
    int part = 0;
    uint32_t part_phase = 0;
    for (int kb = kb_begin; kb < kb_end && ok; ++kb) {
      ok = ptx::mbar_wait(bar_part_full + 8 * part, part_phase, abort_flag, p.status, 0x2400u + part);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      uint32_t v[T::kCols];
      tmem_ld_columns(tmem_base + part * NT + col + (static_cast<uint32_t>(quarter * 32) << 16), v);
      uint64_t s[T::kCols / 2];
#pragma unroll
      for (int j = 0; j < T::kCols / 4; ++j) {
        uint4 raw;
        ptx::ld_shared_v4(scale_base + part * T::kScaleBytes + (col + 4 * j) * 4, raw);
        s[2 * j] = pack_f32x2(raw.x, raw.y);
        s[2 * j + 1] = pack_f32x2(raw.z, raw.w);
      }
      tmem_wait(v);
#pragma unroll
      for (int j = 0; j < T::kCols / 2; ++j) fma_f32x2(acc[j], pack_f32x2(v[2 * j], v[2 * j + 1]), s[j]);
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_part_empty + 8 * part);
      if (++part == kPartials) {
        part = 0;
        part_phase ^= 1u;
      }
    }
  }
  __syncwarp();
  ptx::cluster_wait();
  // Groups of four tokens that a CTA may own; a piece of a group is one 16-byte word per weight row.
  const int groups_each = max(1, (NT / 4) >> split_bits);
  if (warp >= 4 && ok) {
#pragma unroll
    for (int j = 0; j < T::kCols; j += 4) {
      const int group = (col + j) / 4;
      if (4 * group < tokens) {
        const uint32_t dst = ptx::map_to_cta(sums + ((rank * groups_each + (group >> split_bits)) * kBM + row) * 16,
                                             static_cast<uint32_t>(group & (splits - 1)));
        asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(dst), "l"(acc[j / 2]), "l"(acc[j / 2 + 1]) : "memory");
      }
    }
  }
  __syncwarp();
  ptx::cluster_sync();  // all pieces are in place; nobody touches another CTA's memory after this
  // A warp takes 32 weight rows of a group at a time (every warp of the CTA), a lane one row: a column of the result.
  if (*abort_flag == 0) {
    for (int unit = warp;; unit += T::kThreads / 32) {
      const int slot = unit >> 2;
      const int token = 4 * ((slot << split_bits) + rank);
      if (token >= tokens) break;
      const int weight_row = (unit & 3) * 32 + lane;
      const int column = n0 + weight_row;
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int r = 0; r < splits; ++r) {
        uint4 piece;
        ptx::ld_shared_v4(sums + ((r * groups_each + slot) * kBM + weight_row) * 16, piece);
        y[0] += __uint_as_float(piece.x);
        y[1] += __uint_as_float(piece.y);
        y[2] += __uint_as_float(piece.z);
        y[3] += __uint_as_float(piece.w);
      }
      if (column < g.n) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (token + c < tokens) store_one(finish_one(y[c], g, column), g, (m0 + token + c) * g.ldc + column);
        }
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, T::kTmemCols);
  }
}

bool make_map(CUtensorMap* map, const void* base, int elem_bytes, long long rows, long long cols, long long pitch,
              int box_rows, int box_cols) {
  return make_tensormap_2d(map, base, elem_bytes, rows, cols, pitch, box_rows, box_cols, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN, int CTAS, int ACT>
int launch(const GemmFp8& g, cudaStream_t stream) {
  using T = Tile<BN, CTAS>;
  CUtensorMap map_a, map_w;
  if (!make_map(&map_a, g.a, 1, g.m, g.k, g.lda, kBM, kFp8Block)) return LC0B200_ERR_CUDA;
  if (!make_map(&map_w, g.w, 1, g.n, g.k, g.ldw, T::kBRows, kFp8Block)) return LC0B200_ERR_CUDA;
  FpParams p;
  p.g = g;
  p.a_bf16 = nullptr;
  p.ld_a_bf16 = 0;
  // (A TMA store clips a row at whole 16 bytes: with n not a multiple of 8 it would write into the pitch.)
  p.tma_store = g.out_kind == LC0B200_OUT_BF16 && aligned16(g.out) && (g.ldc % 8) == 0 && (g.n % 8) == 0;
  CUtensorMap map_out = map_a;  // placeholder when unused
  if (p.tma_store && !make_map(&map_out, g.out, 2, g.m, g.n, g.ldc, 32, 64)) return LC0B200_ERR_CUDA;
  p.status = device_status_words();
  if (p.status == nullptr) return LC0B200_ERR_CUDA;
  auto kernel = gemm_fp8_kernel<BN, CTAS, ACT>;
  static PerDeviceOnce smem_opt_in;  // per instantiation
  if (allow_dynamic_smem(smem_opt_in, kernel, T::kSmemBytes) != LC0B200_OK) return LC0B200_ERR_CUDA;
  if constexpr (T::kSplitRegs) {
    // A register split that asks for more than the launch has would wait for ever; the 128-wide tile needs none.
    static PerDeviceNumber launch_regs;  // per instantiation
    const DeviceInfo* device = device_info();
    if (device == nullptr) return LC0B200_ERR_CUDA;
    const int regs = ask_once(launch_regs, device->index, [&] {
      cudaFuncAttributes attributes;
      if (cudaFuncGetAttributes(&attributes, kernel) == cudaSuccess) return attributes.numRegs;
      (void)cudaGetLastError();
      return 0;
    });
    if (regs == 0) return LC0B200_ERR_CUDA;
    if (regs < T::kLaunchRegs) return launch<128, 1, ACT>(g, stream);
  }
  const long long tiles = ceil_div_ll(g.m, kBM * CTAS) * ceil_div_ll(g.n, BN);
  const long long max_groups = sm_count() / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((tiles < max_groups ? tiles : max_groups) * CTAS));
  cfg.blockDim = dim3(T::kThreads);
  cfg.dynamicSmemBytes = T::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS == 2 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, map_a, map_w, map_out, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return LC0B200_ERR_CUDA;
  }
  return LC0B200_OK;
}

template <int BN, int CTAS>
int launch(const GemmFp8& g, cudaStream_t stream) {
  switch (g.activation) {
    case LC0B200_ACT_NONE: return launch<BN, CTAS, LC0B200_ACT_NONE>(g, stream);
    case LC0B200_ACT_MISH: return launch<BN, CTAS, LC0B200_ACT_MISH>(g, stream);
    case LC0B200_ACT_RELU: return launch<BN, CTAS, LC0B200_ACT_RELU>(g, stream);
    default: return launch<BN, CTAS, LC0B200_ACT_SWISH>(g, stream);
  }
}

template <int NT, bool BF16_A = false>
int launch_few(const GemmFp8& g, cudaStream_t stream, const bf16* a_bf16 = nullptr, long long ld_a_bf16 = 0) {
  using T = Few<NT>;
  CUtensorMap map_a, map_w;
  if (!make_map(&map_w, g.w, 1, g.n, g.k, g.ldw, kBM, kFp8Block)) return LC0B200_ERR_CUDA;
  map_a = map_w;  // placeholder when unused
  if (!BF16_A && !make_map(&map_a, g.a, 1, g.m, g.k, g.lda, NT, kFp8Block)) return LC0B200_ERR_CUDA;
  FpParams p;
  p.g = g;
  p.tma_store = 0;
  p.a_bf16 = a_bf16;
  p.ld_a_bf16 = ld_a_bf16;
  p.status = device_status_words();
  if (p.status == nullptr) return LC0B200_ERR_CUDA;
  auto kernel = gemm_fp8_few_kernel<NT, BF16_A>;
  static PerDeviceOnce smem_opt_in;  // per instantiation
  if (allow_dynamic_smem(smem_opt_in, kernel, T::kSmemBytes) != LC0B200_OK) return LC0B200_ERR_CUDA;
  // Split k while every CTA stays resident, two to an SM, and has a k block at least.
  const long long tiles = ceil_div_ll(g.n, kBM) * ceil_div_ll(g.m, NT);
  if (tiles > 0x7FFFFFFFLL / kMaxSplits) return LC0B200_ERR_UNSUPPORTED;
  const int k_blocks = static_cast<int>(ceil_div_ll(g.k, kFp8Block));
  int splits = 1;
  while (splits < kMaxSplits && 2 * splits <= k_blocks && tiles * splits <= sm_count()) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
  cfg.blockDim = dim3(T::kThreads);
  cfg.dynamicSmemBytes = T::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, map_w, map_a, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return LC0B200_ERR_CUDA;
  }
  return LC0B200_OK;
}

}  // namespace

// (The Python wrapper counts launches by the same rule.)
bool linear_fp8_few_supported(const GemmFp8& g, const bf16* a, long long lda) {
  return g.m <= 16 && (g.k % 8) == 0 && aligned16(a) && (lda % 8 == 0 || g.m == 1) && aligned16(g.w) && (g.ldw % 16 == 0 || g.n == 1);
}

int linear_fp8_few(const GemmFp8& given, const bf16* a, long long lda, cudaStream_t stream) {
  GemmFp8 g = given;
  if (g.n == 1) g.ldw = ceil_div_ll(g.k, 16) * 16;
  return launch_few<16, true>(g, stream, a, lda);
}

int gemm_fp8(const GemmFp8& given, cudaStream_t stream) {
  GemmFp8 g = given;
  // The pitch of a single row says nothing; make it one that TMA takes.
  if (g.m == 1) g.lda = ceil_div_ll(g.k, 16) * 16;
  if (g.n == 1) g.ldw = ceil_div_ll(g.k, 16) * 16;
  if (!aligned16(g.a) || !aligned16(g.w) || (g.lda % 16) != 0 || (g.ldw % 16) != 0) return gemm_fp8_simt(g, stream);
  // The widest tile that still gives most SMs one; then few-row tiles, the widest that make 60 of them (or the narrowest).
  // (64 rows, 1536 x 1024: 4.2 us on 16-token tiles, 4.6 on 32, 6.3 on 64; 64 rows, 8192 x 8192: 25.6, 18.2, 17.3.)
  const long long enough = sm_count() * 3LL / 5, some = sm_count() * 2LL / 5;
  auto tiles = [&](int rows, int columns) { return ceil_div_ll(g.m, rows) * ceil_div_ll(g.n, columns); };
  if (g.m > 64 && 2 * tiles(2 * kBM, 256) >= enough) return launch<256, 2>(g, stream);
  if (g.m > 64 && tiles(kBM, 128) >= enough) return launch<128, 1>(g, stream);
  if (g.m > 32 && tiles(64, kBM) >= some) return launch_few<64>(g, stream);
  if (g.m > 16 && tiles(32, kBM) >= some) return launch_few<32>(g, stream);
  return launch_few<16>(g, stream);
}

}  // namespace lc0b200
