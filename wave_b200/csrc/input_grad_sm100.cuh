// Input gradient of a frozen MXFP4 linear layer on the tensor cores: dx[M, K] = g[M, N] W[N, K], W = dequant(codes, scales), g bf16.
//
// The scales of W run along K, which is an output dimension here, so the block-scaled MMA does not apply: W is expanded to bf16, which
// holds every E2M1 value times a power of two exactly, and the product runs as kind::f16 with f32 accumulators. 2 M N K flops; for a
// large batch bound by the tensor pipe and, next to it, by shared memory, which a 256 x 256 tile per CTA pair reads and writes at its
// full 128 bytes a clock (per 64 N and CTA: 32 KB written, 32 KB read in 512 clocks).
//
//   warp 0       TMA: g tiles, 128 rows x 64 N, K-major with the 128-byte swizzle
//   warp 1       tcgen05.mma (leader CTA of a pair)
//   warps 2..5   epilogue: accumulator -> bf16 -> dx
//   warps 6..21  expansion of 64 N x 128 K codes a stage within shared memory. A thread takes 32 codes with their one scale. W's rows are
//                contiguous in K, the MMA's N dimension: the tile is an MN-major operand of 64-column groups, rows of 128 bytes per n,
//                swizzled as a TMA load would leave them.
//   warp 22      scales of a stage (four to a row of codes, at any alignment), from global to shared memory
//
// The codes come by TMA, and the scales by a warp of their own, because the expanding threads fence their stores for the tensor core
// (fence.proxy.async), and that fence waits for every load that the thread has in flight: with codes prefetched into registers the kernel
// stood at 480 TFLOP/s, each stage waiting a whole memory latency.
//
// With few tiles the sum over N is cut into slices: one cluster of `slices` pairs (or CTAs) to a tile, which then add their f32 accumulators
// through distributed shared memory, in slice order, each its share of the rows. No workspace, no second launch, the same bits on every run.
//
// CG = 2: 256 x 256 tiles, each CTA holds 128 rows of g and expands 128 columns of W; CG = 1: 128 x 128 tiles. Both accumulators of
// neighbouring tiles are in tensor memory, so an epilogue runs under the next tile's products.
//
// 8192^3 in a graph of launches: 793 to 832 us by board, 1322 to 1386 TFLOP/s, at the power limit (cuBLAS' bf16 product sustains 1368); a call among others
// on changing inputs 911 to 926 us, about 1200 TFLOP/s. 600 x 4000 x 2048 24 us, of which 13 are its 32 steps.
#pragma once
#include "ptx.cuh"

namespace wb {

template <int CG>
struct InputGradCfg {
  static constexpr int BM = 128;          // rows of a CTA
  static constexpr int BN = 64;           // contraction per stage
  static constexpr int COLS = 128;        // columns of W that a CTA expands
  static constexpr int TILE_K = COLS * CG;
  static constexpr int A_BYTES = BM * BN * 2;
  static constexpr int B_BYTES = COLS * BN * 2;
  static constexpr int A_STAGES = 6;                 // deeper than B's: a load from memory takes longer than an expansion
  static constexpr int B_STAGES = 6;
  static constexpr int CODE_BYTES = COLS / 2 * BN;   // of a stage
  static constexpr int SCALE_BYTES = COLS / 32 * BN;
  static constexpr int CODE_STAGES = 6;
  static constexpr int SCALE_BATCH = 8;              // stages whose scales are loaded together; two batches in shared memory
  static constexpr int SUM_PITCH = TILE_K * 4 + 16;  // rows of f32 accumulators in shared memory; 16 bytes spread the lanes over the banks
  static constexpr int TMEM_COLS = 2 * TILE_K;
  static constexpr int NUM_BARRIERS = 2 * (A_STAGES + B_STAGES + CODE_STAGES) + 8;
  static constexpr int B_BASE = A_STAGES * A_BYTES;
  static constexpr int CODE_BASE = B_BASE + B_STAGES * B_BYTES;
  static constexpr int SCALE_BASE = CODE_BASE + CODE_STAGES * CODE_BYTES;
  static constexpr int BAR_BASE = SCALE_BASE + 2 * SCALE_BATCH * SCALE_BYTES;
  static constexpr int SMEM_BYTES = BAR_BASE + NUM_BARRIERS * 8 + 16 + 1024;
  static constexpr int EXPAND_WARPS = 16;
  static constexpr int GROUPS = 4;                   // of the expanding warps, each on a stage of its own
  static constexpr int GROUP_WARPS = EXPAND_WARPS / GROUPS;
  static_assert(GROUPS <= B_STAGES && GROUPS <= SCALE_BATCH && EXPAND_WARPS % GROUPS == 0, "a group moves on by less than a ring");
  static constexpr int THREADS = (7 + EXPAND_WARPS) * 32;
  static_assert(SMEM_BYTES >= kSmemOfTmemKernel, "keeps other kernels with tensor memory off the SM");
  static_assert(CODE_BASE % 1024 == 0 && CODE_BYTES % 1024 == 0 && BAR_BASE % 8 == 0 && BM * SUM_PITCH <= CODE_BASE && SMEM_BYTES <= 227 * 1024, "shared memory");
};

struct InputGradParams {
  const uint8_t* scales;  // [N, K/32], pitch ld_scales
  __nv_bfloat16* dx;
  long long ld_scales, ldd;
  int M, N, K, tiles_m, tiles_k, group_k, slices;
  int scale_words;  // four scales of a row are an aligned word (K % 128 == 0)
  int* status;
};

// Instruction descriptor of kind::f16: f32 accumulator, bf16 operands, A K-major, B MN-major.
__host__ __device__ constexpr uint32_t make_idesc_bf16_bt(int m, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// MN-major operand with the 128-byte swizzle: 64 elements of MN to a row of 128 bytes, one row per k, 8 rows (1024 bytes) to the swizzle's
// period along k; the next 64 elements of MN follow `mn_stride` bytes on.
__device__ __forceinline__ uint64_t make_desc_mn_sw128(uint32_t smem_addr, uint32_t mn_stride) {
  uint64_t d = 0;
  d |= uint64_t((smem_addr & 0x3FFFFu) >> 4);
  d |= uint64_t(mn_stride >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrival on the leader's barrier for operand bytes that lie in THIS CTA's shared memory: the pair's MMA reads them through this SM's own tensor
// core, so the stores have to be complete here before the signal leaves (every writer has executed fence.proxy.async, the warp has met), which a
// release at CTA scope orders. At cluster scope the release waits for a round trip through the memory system, about 2 us a stage under
// load: 8192 x 4096 x 4096 275 against 208 us.
__device__ __forceinline__ void mbar_arrive_own_operand(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// The barrier at this offset in every CTA of the pair completes once the MMAs issued so far have.
template <int CG>
__device__ __forceinline__ void tc_commit_all(uint32_t bar, uint16_t pair_mask) {
  if constexpr (CG == 1)
    tc_commit<1>(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(pair_mask)
                 : "memory");
}

// 2^(s - 127) twice as a bf16 pair; exact for every E8M0 value (2^-127 is a bf16 subnormal), NaN for 255.
__device__ __forceinline__ uint32_t e8m0_bf16x2(uint32_t s) {
  const uint32_t h = s == 255u ? 0x7fffu : s == 0u ? 0x0040u : s << 7;
  return h | h << 16;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Four E2M1 codes (16 bits) times a scale as two bf16 pairs. The magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 are looked up by byte permutes,
// high bytes and low bytes apart; bit 3 of a code is the sign.
__device__ __forceinline__ void expand4(uint32_t w, uint32_t scale, uint32_t& lo_pair, uint32_t& hi_pair) {
  const uint32_t sel = w & 0x7777u;
  const uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);
  const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, sel);
  const uint32_t p0 = __byte_perm(lo, hi, 0x5140) | ((w << 12) & 0x8000u) | ((w << 24) & 0x80000000u);
  const uint32_t p1 = __byte_perm(lo, hi, 0x7362) | ((w << 4) & 0x8000u) | ((w << 16) & 0x80000000u);
  lo_pair = mul_bf16x2(p0, scale);
  hi_pair = mul_bf16x2(p1, scale);
}

// A CTA's share of the rows of a tile, added up over the slices: eight columns a thread, the loads of all slices in flight together.
template <int CG, int S>
__device__ __forceinline__ void sum_slices(const InputGradParams& p, uint32_t smem_base, int mt, int kt, int rank, int slice) {
  using Cfg = InputGradCfg<CG>;
  const int first = Cfg::BM * slice / S, rows = Cfg::BM * (slice + 1) / S - first;
  constexpr int ITEMS = S == 2 ? 3 : S == 3 ? 2 : 1;  // pieces of a thread in flight: what registers there are hold
  for (int e0 = threadIdx.x; e0 < rows * (Cfg::TILE_K / 8); e0 += ITEMS * Cfg::THREADS) {
    float v[ITEMS][S][8];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = e0 + i * Cfg::THREADS;
      if (ITEMS > 1 && e >= rows * (Cfg::TILE_K / 8)) break;
      const int in = first + e / (Cfg::TILE_K / 8), c = e % (Cfg::TILE_K / 8) * 8;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t at = mapa_shared(smem_base + uint32_t(in) * Cfg::SUM_PITCH + c * 4, uint32_t(s * CG + rank));
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[i][s][4 * h]), "=f"(v[i][s][4 * h + 1]), "=f"(v[i][s][4 * h + 2]), "=f"(v[i][s][4 * h + 3])
                       : "r"(at + 16 * h));
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = e0 + i * Cfg::THREADS;
      if (ITEMS > 1 && e >= rows * (Cfg::TILE_K / 8)) break;
      const int row = (mt * CG + rank) * Cfg::BM + first + e / (Cfg::TILE_K / 8), col = kt * Cfg::TILE_K + e % (Cfg::TILE_K / 8) * 8;
      if (row >= p.M || col >= p.K) continue;
      float sum[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] = v[i][0][j];
#pragma unroll
        for (int s = 1; s < S; ++s) sum[j] += v[i][s][j];
      }
      if (WB_CHECK(row < p.M && col + 8 <= p.K, kCheckOutputIndex, (long long)row << 32 | col))
        *reinterpret_cast<uint4*>(p.dx + (long long)row * p.ldd + col) = make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]),
                                                                                    pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
    }
  }
}

template <int CG>
__global__ void __launch_bounds__(InputGradCfg<CG>::THREADS, 1)
input_grad_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_codes, const InputGradParams p) {
  using Cfg = InputGradCfg<CG>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = (CG == 2 || p.slices > 1) ? cluster_ctarank() : 0u;
  const uint32_t rank = cluster_rank % CG;         // in the pair
  const uint32_t leader_rank = cluster_rank - rank;  // of the pair's leader in the cluster
  const bool leader = rank == 0;
  const int slice = int(cluster_rank) / CG;

  const uint32_t bar_base = smem_base + Cfg::BAR_BASE;
  auto a_full = [&](int s) { return bar_base + 8u * s; };
  auto a_empty = [&](int s) { return bar_base + 8u * (Cfg::A_STAGES + s); };
  constexpr int B0 = 2 * Cfg::A_STAGES, C0 = B0 + 2 * Cfg::B_STAGES, D0 = C0 + 2 * Cfg::CODE_STAGES;
  auto b_full = [&](int s) { return bar_base + 8u * (B0 + s); };
  auto b_empty = [&](int s) { return bar_base + 8u * (B0 + Cfg::B_STAGES + s); };
  auto code_full = [&](int s) { return bar_base + 8u * (C0 + s); };
  auto code_empty = [&](int s) { return bar_base + 8u * (C0 + Cfg::CODE_STAGES + s); };
  auto acc_full = [&](int s) { return bar_base + 8u * (D0 + s); };
  auto acc_empty = [&](int s) { return bar_base + 8u * (D0 + 2 + s); };
  auto scale_full = [&](int s) { return bar_base + 8u * (D0 + 4 + s); };
  auto scale_empty = [&](int s) { return bar_base + 8u * (D0 + 6 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + Cfg::BAR_BASE + Cfg::NUM_BARRIERS * 8);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  WaitCtx ctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::A_STAGES; ++s) {
      mbar_init(a_full(s), 1);
      mbar_init(a_empty(s), 1);
    }
    for (int s = 0; s < Cfg::B_STAGES; ++s) {
      mbar_init(b_full(s), Cfg::GROUP_WARPS * CG);
      mbar_init(b_empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full(s), 1);
      mbar_init(acc_empty(s), 4 * CG);
    }
    for (int s = 0; s < Cfg::CODE_STAGES; ++s) {
      mbar_init(code_full(s), 1);
      mbar_init(code_empty(s), Cfg::GROUP_WARPS);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(scale_full(s), 1);
      mbar_init(scale_empty(s), Cfg::EXPAND_WARPS);
    }
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<CG>(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<CG>();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&map_g);
    prefetch_tensormap(&map_codes);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (CG == 2 || p.slices > 1) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  const int num_tiles = p.tiles_m * p.tiles_k;
  const int first_tile = blockIdx.x / (CG * p.slices), tile_step = gridDim.x / (CG * p.slices);  // with slices: one tile per cluster
  const int all_steps = (p.N + Cfg::BN - 1) / Cfg::BN;
  const int step0 = int((long long)all_steps * slice / p.slices);
  const int steps = int((long long)all_steps * (slice + 1) / p.slices) - step0;  // at least one
  // tiles in groups of group_k columns of tiles, each swept down the rows
  auto tile_at = [&](int tile, int& mt, int& kt) {
    const int per = p.group_k * p.tiles_m;
    const int group = tile / per, in = tile - group * per;
    const int width = min(p.group_k, p.tiles_k - group * p.group_k);
    mt = in / width;
    kt = group * p.group_k + in - mt * width;
  };

  if (warp == 0) {
    uint32_t stage = 0, phase = 0, cs = 0, cphase = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      int mt, kt;
      tile_at(tile, mt, kt);
      const int row = (mt * CG + int(rank)) * Cfg::BM;
      const int col = kt * Cfg::TILE_K + int(rank) * Cfg::COLS;
      for (int s = 0; s < steps; ++s) {
        if (!mbar_wait(code_empty(cs), cphase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;  // given up: nothing more is issued
        if (elect_one()) {
          mbar_expect_tx(code_full(cs), Cfg::CODE_BYTES);
          tma_load_2d<CG>(smem_base + Cfg::CODE_BASE + cs * Cfg::CODE_BYTES, &map_codes, col / 2, (step0 + s) * Cfg::BN, code_full(cs));
        }
        __syncwarp();
        if (++cs == Cfg::CODE_STAGES) { cs = 0; cphase ^= 1u; }
        if (!mbar_wait(a_empty(stage), phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;
        const uint32_t bar = CG == 2 ? mapa_shared(a_full(stage), leader_rank) : a_full(stage);
        if (elect_one()) {
          if (leader) mbar_expect_tx(a_full(stage), Cfg::A_BYTES * CG);
          tma_load_2d<CG>(smem_base + stage * Cfg::A_BYTES, &map_g, (step0 + s) * Cfg::BN, row, bar);
        }
        __syncwarp();
        if (++stage == Cfg::A_STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    pdl_launch_dependents();
  } else if (warp == 1) {
    if (leader) {
      const uint32_t idesc = make_idesc_bf16_bt(Cfg::BM * CG, Cfg::TILE_K);
      const uint16_t pair_mask = uint16_t(3u << leader_rank);
      uint32_t as = 0, aphase = 0, bs = 0, bphase = 0;
      int it = 0;
      for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++it) {
        const int acc = it & 1;
        if (it >= 2) mbar_wait<CG == 2>(acc_empty(acc), uint32_t((it - 2) >> 1) & 1u, ctx, WB_DEV_TIMEOUT_MMA_ACC);
        tc_fence_after_sync();
        const uint32_t d = tmem_base + acc * Cfg::TILE_K;
        for (int s = 0; s < steps; ++s) {
          mbar_wait(a_full(as), aphase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
          mbar_wait<CG == 2>(b_full(bs), bphase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
          tc_fence_after_sync();
          const uint64_t a_desc = make_desc_k_sw128(smem_base + as * Cfg::A_BYTES);
          const uint64_t b_desc = make_desc_mn_sw128(smem_base + Cfg::B_BASE + bs * Cfg::B_BYTES, Cfg::BN * 128);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < Cfg::BN / 16; ++k)  // 16 n: 32 bytes along A's rows, two groups of eight rows of B
              mma_f16<CG>(d, a_desc + uint64_t(k * 2), b_desc + uint64_t(k * (2048 >> 4)), idesc, (s > 0 || k > 0) ? 1u : 0u);
            tc_commit_all<CG>(b_empty(bs), pair_mask);
            tc_commit_all<CG>(a_empty(as), pair_mask);
            if (s == steps - 1) tc_commit_all<CG>(acc_full(acc), pair_mask);
          }
          __syncwarp();
          if (++as == Cfg::A_STAGES) { as = 0; aphase ^= 1u; }
          if (++bs == Cfg::B_STAGES) { bs = 0; bphase ^= 1u; }
        }
      }
    }
  } else if (warp < 6) {
    const int quad = warp & 3;
    int it = 0;
    if (p.slices == 1)
    for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++it) {
      int mt, kt;
      tile_at(tile, mt, kt);
      const int as = it & 1;
      mbar_wait(acc_full(as), uint32_t(it >> 1) & 1u, ctx, WB_DEV_TIMEOUT_EPILOGUE);
      tc_fence_after_sync();
      const int row = (mt * CG + int(rank)) * Cfg::BM + quad * 32 + (lane & ~3);  // of this lane's first store
      __nv_bfloat16* dst = p.dx + (long long)row * p.ldd + (lane & 3) * 8;
      const long long pitch = p.ldd / 8;
#pragma unroll 1
      for (int c = 0; c < Cfg::TILE_K; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + (uint32_t(quad * 32) << 16) + as * Cfg::TILE_K + c, r);
        tmem_ld_wait();
        const int col = kt * Cfg::TILE_K + c;
        if (col >= p.K) break;  // K is a multiple of 32
        // Four neighbouring lanes exchange their rows' four pieces of 8 columns, so that a store writes 64 consecutive bytes of each of 8 rows
        // (6826 x 256 x 5216, mostly epilogue: 47.5 us with a row to a lane, 37.3)
        uint32_t q[4][4];
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j / 4][j % 4] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j & o) continue;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, (lane & o) ? q[j][w] : q[j | o][w], o);
              if (lane & o) q[j][w] = got;
              else q[j | o][w] = got;
            }
          }
        uint4* at = reinterpret_cast<uint4*>(dst + col);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (row + j < p.M && WB_CHECK(col + (lane & 3) * 8 + 8 <= p.K, kCheckOutputIndex, (long long)(row + j) << 32 | col)) at[j * pitch] = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster_relaxed(mapa_shared(acc_empty(as), leader_rank));  // publishes no data: the reads are complete
        else mbar_arrive(acc_empty(as));
      }
    }
  } else if (warp < 6 + Cfg::EXPAND_WARPS) {
    // 32 codes at a time: row n of the stage, block of 32 columns. Eight lanes of neighbouring n read and write at a time: the swizzles (64 bytes
    // of the codes, 128 of the operand) put their 16-byte pieces into different banks. A stage is a chain of waits, so that the warps work
    // in groups, each on every GROUPS-th stage.
    const int group = (warp - 6) / Cfg::GROUP_WARPS;
    const int id0 = ((warp - 6) % Cfg::GROUP_WARPS) * 32 + lane;
    const int my_tiles = first_tile < num_tiles ? (num_tiles - first_tile + tile_step - 1) / tile_step : 0;
    const long long total = (long long)my_tiles * steps;
    uint32_t stage = group, phase = 0;
    for (long long i = group; i < total; i += Cfg::GROUPS) {
      const int at = int(i & (2 * Cfg::SCALE_BATCH - 1)), half = at / Cfg::SCALE_BATCH, in_batch = at & (Cfg::SCALE_BATCH - 1);
      const int cs = int(i % Cfg::CODE_STAGES);
      if (in_batch < Cfg::GROUPS) mbar_wait(scale_full(half), uint32_t(i / (2 * Cfg::SCALE_BATCH)) & 1u, ctx, WB_DEV_TIMEOUT_MMA_FULL);
      mbar_wait(code_full(cs), uint32_t(i / Cfg::CODE_STAGES) & 1u, ctx, WB_DEV_TIMEOUT_MMA_FULL);
      constexpr int ITEMS = Cfg::BN * 4 / (Cfg::GROUP_WARPS * 32);
      uint32_t v[ITEMS][16];
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) {
        const int id = id0 + u * Cfg::GROUP_WARPS * 32;
        const int n = (id & 7) + 8 * (id >> 5), blk = (id >> 3) & 3;
        uint32_t word[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(word[0]), "=r"(word[1]), "=r"(word[2]), "=r"(word[3])
                     : "r"(smem_base + Cfg::CODE_BASE + cs * Cfg::CODE_BYTES + n * 64 + ((blk ^ ((n >> 1) & 3)) << 4)));
        const uint32_t f = e8m0_bf16x2(smem_gen[Cfg::SCALE_BASE + at * Cfg::SCALE_BYTES + n * 4 + blk]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          expand4(word[q], f, v[u][4 * q], v[u][4 * q + 1]);
          expand4(word[q] >> 16, f, v[u][4 * q + 2], v[u][4 * q + 3]);
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(code_empty(cs));
        if (in_batch >= Cfg::SCALE_BATCH - Cfg::GROUPS) mbar_arrive(scale_empty(half));
      }
      mbar_wait(b_empty(stage), phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER);  // only now: a stage is held for the stores alone
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) {
        const int id = id0 + u * Cfg::GROUP_WARPS * 32;
        const int n = (id & 7) + 8 * (id >> 5), blk = (id >> 3) & 3;
        const uint32_t to = smem_base + Cfg::B_BASE + stage * Cfg::B_BYTES + (blk >> 1) * (Cfg::BN * 128) + n * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + ((((blk & 1) * 4 + q) ^ (n & 7)) << 4)), "r"(v[u][4 * q]),
                       "r"(v[u][4 * q + 1]), "r"(v[u][4 * q + 2]), "r"(v[u][4 * q + 3])
                       : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_own_operand(mapa_shared(b_full(stage), leader_rank));
        else mbar_arrive(b_full(stage));
      }
      stage += Cfg::GROUPS;
      if (stage >= Cfg::B_STAGES) { stage -= Cfg::B_STAGES; phase ^= 1u; }
    }
  } else {
    // scales of rows `lane` and `lane + 32` of a stage, four to a row: the loads of a batch of stages are in flight together, while the batch before
    // is being read
    const int my_tiles = first_tile < num_tiles ? (num_tiles - first_tile + tile_step - 1) / tile_step : 0;
    const long long total = (long long)my_tiles * steps;
    int tile = first_tile, s = 0, col = 0;
    for (long long i = 0; i < total; i += Cfg::SCALE_BATCH) {
      uint32_t word[Cfg::SCALE_BATCH][2];
#pragma unroll
      for (int j = 0; j < Cfg::SCALE_BATCH; ++j) {
        if (s == 0 && i + j < total) {
          int mt, kt;
          tile_at(tile, mt, kt);
          col = (kt * Cfg::TILE_K + int(rank) * Cfg::COLS) / 32;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = (step0 + s) * Cfg::BN + lane + 32 * h;
          const bool real = i + j < total && row < p.N;
          const uint8_t* at = p.scales + row * p.ld_scales + col;
          word[j][h] = 0x7f7f7f7fu;
          if (p.scale_words) {
            if (real && col * 32 < p.K) word[j][h] = *reinterpret_cast<const uint32_t*>(at);
          } else {
            uint32_t w = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) w |= uint32_t(real && (col + b) * 32 < p.K ? at[b] : 0x7fu) << (8 * b);
            word[j][h] = w;
          }
        }
        if (++s == steps) { s = 0; tile += tile_step; }
      }
      const int half = int(i / Cfg::SCALE_BATCH) & 1;
      mbar_wait(scale_empty(half), (uint32_t(i / (2 * Cfg::SCALE_BATCH)) & 1u) ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER);
      uint32_t* dst = reinterpret_cast<uint32_t*>(smem_gen + Cfg::SCALE_BASE + half * Cfg::SCALE_BATCH * Cfg::SCALE_BYTES);
#pragma unroll
      for (int j = 0; j < Cfg::SCALE_BATCH; ++j) {
        dst[j * Cfg::BN + lane] = word[j][0];
        dst[j * Cfg::BN + lane + 32] = word[j][1];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(scale_full(half));
    }
  }

  if (p.slices > 1) {
    // the one accumulator into this CTA's shared memory, whose stages are all read once it is complete: 32 columns at a time, the expanding
    // warps help
    if (warp >= 2 && warp < 6 + Cfg::EXPAND_WARPS) {
      mbar_wait(acc_full(0), 0u, ctx, WB_DEV_TIMEOUT_EPILOGUE);
      tc_fence_after_sync();
      const int quad = warp & 3;
#pragma unroll 1
      for (int c = (warp - 2) / 4 * 32; c < Cfg::TILE_K; c += (4 + Cfg::EXPAND_WARPS) / 4 * 32) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + (uint32_t(quad * 32) << 16) + c, r);
        tmem_ld_wait();
        const uint32_t at = smem_base + uint32_t(quad * 32 + lane) * Cfg::SUM_PITCH + c * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + 16 * j), "r"(r[4 * j]), "r"(r[4 * j + 1]), "r"(r[4 * j + 2]), "r"(r[4 * j + 3])
                       : "memory");
      }
      tc_fence_before_sync();
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    int mt, kt;
    tile_at(first_tile, mt, kt);
    switch (p.slices) {
      case 2: sum_slices<CG, 2>(p, smem_base, mt, kt, int(rank), slice); break;
      case 3: sum_slices<CG, 3>(p, smem_base, mt, kt, int(rank), slice); break;
      case 4: sum_slices<CG, 4>(p, smem_base, mt, kt, int(rank), slice); break;
      default:
        if constexpr (CG == 1) {
          if (p.slices == 8) sum_slices<CG, 8>(p, smem_base, mt, kt, int(rank), slice);
          else sum_slices<CG, 6>(p, smem_base, mt, kt, int(rank), slice);
        }
    }
  }

  // nobody leaves while the other CTA's barriers may still be signalled or its operands read
  tc_fence_before_sync();
  __syncthreads();
  if (CG == 2 || p.slices > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<CG>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace wb
