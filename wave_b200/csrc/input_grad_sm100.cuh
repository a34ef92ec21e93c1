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
//   warps 6..13  expansion: 64 N x 128 K codes a stage, from global memory (three stages ahead, in registers) to shared memory. A thread
//                takes 32 codes with their one scale. W's rows are contiguous in K, the MMA's N dimension: the tile is an MN-major
//                operand of 64-column groups, rows of 128 bytes per n, swizzled as a TMA load would leave them.
//
// CG = 2: 256 x 256 tiles, each CTA holds 128 rows of g and expands 128 columns of W; CG = 1: 128 x 128 tiles. Both accumulators of
// neighbouring tiles are in tensor memory, so an epilogue runs under the next tile's products.
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
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int TMEM_COLS = 2 * TILE_K;
  static constexpr int NUM_BARRIERS = 3 * STAGES + 4;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + NUM_BARRIERS * 8 + 16 + 1024;
  static constexpr int EXPAND_WARPS = 8;
  static constexpr int THREADS = (6 + EXPAND_WARPS) * 32;
};

struct InputGradParams {
  const uint8_t* codes;   // [N, K/2]
  const uint8_t* scales;  // [N, K/32], pitch ld_scales
  __nv_bfloat16* dx;
  long long ld_scales, ldd;
  int M, N, K, tiles_m, tiles_k, group_k;
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

template <int CG>
__global__ void __launch_bounds__(InputGradCfg<CG>::THREADS, 1)
input_grad_kernel(const __grid_constant__ CUtensorMap map_g, const InputGradParams p) {
  using Cfg = InputGradCfg<CG>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;

  const uint32_t bar_base = smem_base + STAGES * Cfg::STAGE_BYTES;
  auto a_full = [&](int s) { return bar_base + 8u * s; };
  auto b_full = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto empty_bar = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };
  auto acc_full = [&](int s) { return bar_base + 8u * (3 * STAGES + s); };
  auto acc_empty = [&](int s) { return bar_base + 8u * (3 * STAGES + 2 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + STAGES * Cfg::STAGE_BYTES + Cfg::NUM_BARRIERS * 8);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  WaitCtx ctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(a_full(s), 1);
      mbar_init(b_full(s), Cfg::EXPAND_WARPS * CG);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full(s), 1);
      mbar_init(acc_empty(s), 4 * CG);
    }
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<CG>(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<CG>();
  }
  if (warp == 0 && lane == 0) prefetch_tensormap(&map_g);
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  const int num_tiles = p.tiles_m * p.tiles_k;
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;
  const int steps = (p.N + Cfg::BN - 1) / Cfg::BN;
  // tiles in groups of group_k columns of tiles, each swept down the rows
  auto tile_at = [&](int tile, int& mt, int& kt) {
    const int per = p.group_k * p.tiles_m;
    const int group = tile / per, in = tile - group * per;
    const int width = min(p.group_k, p.tiles_k - group * p.group_k);
    mt = in / width;
    kt = group * p.group_k + in - mt * width;
  };

  if (warp == 0) {
    uint32_t stage = 0, phase = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      int mt, kt;
      tile_at(tile, mt, kt);
      const int row = (mt * CG + int(rank)) * Cfg::BM;
      for (int s = 0; s < steps; ++s) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;  // given up: nothing more is issued
        const uint32_t bar = CG == 2 ? mapa_shared(a_full(stage), 0) : a_full(stage);
        if (elect_one()) {
          if (leader) mbar_expect_tx(a_full(stage), Cfg::A_BYTES * CG);
          tma_load_2d<CG>(smem_base + stage * Cfg::STAGE_BYTES, &map_g, s * Cfg::BN, row, bar);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    pdl_launch_dependents();
  } else if (warp == 1) {
    if (leader) {
      const uint32_t idesc = make_idesc_bf16_bt(Cfg::BM * CG, Cfg::TILE_K);
      const uint32_t peer_empty = CG == 2 ? mapa_shared(empty_bar(0), 1) : 0u;
      const uint32_t peer_acc_full = CG == 2 ? mapa_shared(acc_full(0), 1) : 0u;
      uint32_t stage = 0, phase = 0;
      int it = 0;
      for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++it) {
        const int as = it & 1;
        if (it >= 2) mbar_wait<CG == 2>(acc_empty(as), uint32_t((it - 2) >> 1) & 1u, ctx, WB_DEV_TIMEOUT_MMA_ACC);
        tc_fence_after_sync();
        const uint32_t d = tmem_base + as * Cfg::TILE_K;
        for (int s = 0; s < steps; ++s) {
          mbar_wait(a_full(stage), phase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
          mbar_wait<CG == 2>(b_full(stage), phase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
          tc_fence_after_sync();
          const uint32_t sA = smem_base + stage * Cfg::STAGE_BYTES;
          const uint64_t a_desc = make_desc_k_sw128(sA);
          const uint64_t b_desc = make_desc_mn_sw128(sA + Cfg::A_BYTES, Cfg::BN * 128);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < Cfg::BN / 16; ++k)  // 16 n: 32 bytes along A's rows, two groups of eight rows of B
              mma_f16<CG>(d, a_desc + uint64_t(k * 2), b_desc + uint64_t(k * (2048 >> 4)), idesc, (s > 0 || k > 0) ? 1u : 0u);
            tc_commit<CG>(empty_bar(stage));
            if constexpr (CG == 2) tc_commit<CG>(peer_empty + 8u * stage);
            if (s == steps - 1) {
              tc_commit<CG>(acc_full(as));
              if constexpr (CG == 2) tc_commit<CG>(peer_acc_full + 8u * as);
            }
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp < 6) {
    const int quad = warp & 3;
    int it = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++it) {
      int mt, kt;
      tile_at(tile, mt, kt);
      const int as = it & 1;
      mbar_wait(acc_full(as), uint32_t(it >> 1) & 1u, ctx, WB_DEV_TIMEOUT_EPILOGUE);
      tc_fence_after_sync();
      const int row = (mt * CG + int(rank)) * Cfg::BM + quad * 32 + lane;
      __nv_bfloat16* dst = p.dx + (long long)row * p.ldd;
#pragma unroll 1
      for (int c = 0; c < Cfg::TILE_K; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + (uint32_t(quad * 32) << 16) + as * Cfg::TILE_K + c, r);
        tmem_ld_wait();
        const int col = kt * Cfg::TILE_K + c;
        if (row < p.M && col < p.K) {  // K is a multiple of 32
          uint4* q = reinterpret_cast<uint4*>(dst + col);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            q[j] = make_uint4(pack_bf16x2(__uint_as_float(r[8 * j]), __uint_as_float(r[8 * j + 1])),
                              pack_bf16x2(__uint_as_float(r[8 * j + 2]), __uint_as_float(r[8 * j + 3])),
                              pack_bf16x2(__uint_as_float(r[8 * j + 4]), __uint_as_float(r[8 * j + 5])),
                              pack_bf16x2(__uint_as_float(r[8 * j + 6]), __uint_as_float(r[8 * j + 7])));
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(mapa_shared(acc_empty(as), 0));
        else mbar_arrive(acc_empty(as));
      }
    }
  } else {
    // a thread's 32 codes: row n of the stage, block of 32 columns
    const int id = (warp - 6) * 32 + lane;
    const int n = (id & 7) + 8 * (id >> 5), blk = (id >> 3) & 3;
    const uint32_t row_at = uint32_t((blk >> 1) * (Cfg::BN * 128) + n * 128);
    const uint32_t chunk0 = uint32_t((blk & 1) * 4), flip = uint32_t(n & 7);
    uint32_t stage = 0, phase = 0;
    int tile = first_tile, s = 0;  // of the next load
    uint4 codes[3];
    uint32_t scale[3];
    int col = 0;
    auto fetch = [&](uint4& c, uint32_t& e) {
      c = make_uint4(0u, 0u, 0u, 0u);
      e = 127u;
      if (tile >= num_tiles) return;
      if (s == 0) {
        int mt, kt;
        tile_at(tile, mt, kt);
        col = kt * Cfg::TILE_K + int(rank) * Cfg::COLS + blk * 32;
      }
      const int row = s * Cfg::BN + n;
      if (row < p.N && col < p.K) {
        c = *reinterpret_cast<const uint4*>(p.codes + (long long)row * (p.K / 2) + col / 2);
        e = p.scales[row * p.ld_scales + col / 32];
      }
      if (++s == steps) { s = 0; tile += tile_step; }
    };
    const int my_tiles = first_tile < num_tiles ? (num_tiles - first_tile + tile_step - 1) / tile_step : 0;
    const long long total = (long long)my_tiles * steps;
#pragma unroll
    for (int i = 0; i < 3; ++i) fetch(codes[i], scale[i]);
    for (long long i = 0; i < total; ++i) {
      const uint4 c = codes[0];
      const uint32_t f = e8m0_bf16x2(scale[0]);
      codes[0] = codes[1]; scale[0] = scale[1];
      codes[1] = codes[2]; scale[1] = scale[2];
      fetch(codes[2], scale[2]);
      mbar_wait(empty_bar(stage), phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER);
      const uint32_t sB = smem_base + stage * Cfg::STAGE_BYTES + Cfg::A_BYTES + row_at;
      const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t v[4];
        expand4(word[q], f, v[0], v[1]);
        expand4(word[q] >> 16, f, v[2], v[3]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sB + (((chunk0 + q) ^ flip) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                     : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(mapa_shared(b_full(stage), 0));
        else mbar_arrive(b_full(stage));
      }
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    }
  }

  // nobody leaves while the other CTA's barriers may still be signalled or its operands read
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<CG>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace wb
