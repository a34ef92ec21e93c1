// Low-rank adapters of many requests beside a shared projection, forward and backward:
//
//   out[t] = y[t] + s_l B_l (A_l x[t])        l = ids[t], A_l [R, K], B_l [N, R], bf16; rows without an adapter keep y
//   u[t]   = s_l B_l^T g[t]      dx[t] = A_l^T u[t]      dA_l = sum_t u[t] x[t]^T      dB_l = s_l sum_t g[t] (A_l x[t])^T
//
// Three kernels: `shrink` (rows times a wide matrix onto the ranks: A_l x, B_l^T g), `expand` (ranks onto wide rows: B_l h, A_l^T u) and
// `outer` (sums over the rows of an adapter). At the ranks adapters have (2 R flops per two bytes of x) they are bound by HBM for many rows and by latency
// for few, and what counts is that every row of x, y and g moves once, in whole 32-byte sectors, with enough of them in flight.
//
// shrink and expand come in three forms each, chosen by rules on rows, ranks, types and alignment (few_rows, wide_shrink and wide_expand in adapt.cu):
//   few    up to 64 rows with few rows to an adapter: operands from global memory straight to registers, every warp finds the rows of its adapter itself
//          by a vote, no barrier before the first load; f32 FMAs in the second product.
//   tile   mma.sync, at any alignment and rank: rows are taken in chunks of 64 neighbours, every CTA sorts the chunk's rows by adapter itself (64 compares a
//          thread; a chunk of one sequence is noticed and not sorted), so that no launch precedes it and ids need no order.
//   wide   tcgen05 with tiles by TMA, for aligned bf16 rows: shrink from 2048 rows or above 32 ranks, expand at 33 to 64 ranks where y and out are larger
//          than L2. mma.sync is slower there: `expand` with its three bf16 parts 97 against 57 us at rank 64, 8192 rows and 8192 columns.
// outer is mma.sync at every size.
//
// Layouts for mma.sync m16n8k16: an MMA adds over its 16 k in any order, so a lane may hold any 8 consecutive k of a row (one 16-byte load, two
// MMAs) as long as the other operand is permuted alike, and the columns of an output tile may be dealt to the lanes so that each has 8
// neighbours. Operands whose contraction runs down the rows of memory (B_l^T, A_l^T, the outer products) are transposed by byte permutes of
// two registers, or by ldmatrix where they come through shared memory.
//
// The hidden vector h = s_l A_l x (R numbers a row) is f32, in memory too. The second product takes it as three bf16 parts, 8 bits of its significand
// each, which add up to it exactly: nothing of an f32 sum is lost on the way, whatever the result's type. Two parts (17 bits) would save a third of
// that product's MMAs, and show in a result whose y cancels most of what the adapter adds.
//
// Dependent launches: shrink and outer touch memory only once the kernel before them is complete. expand is always launched behind a shrink, which lets it
// begin after that point: what it reads before its own wait (y, w, ids) is older than the shrink, and it writes nothing before it.
#pragma once
#include <cuda_bf16.h>

#include "checks.cuh"
#include "input_grad_sm100.cuh"
#include "ptx.cuh"

namespace wb {

constexpr int kChunkRows = 64;
constexpr int kAdapterWarps = 8;
constexpr int kAdapterThreads = kAdapterWarps * 32;
constexpr int kExpandCols = 32;  // columns of a warp's tile

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// COUNT consecutive bf16 as registers; `whole`: one aligned vector load, otherwise the first `valid` of them one by one, zeros behind.
template <int COUNT>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16* p, bool whole, int valid, uint32_t (&r)[COUNT / 2]) {
  if (whole) {
    if constexpr (COUNT == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
    } else if constexpr (COUNT == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      r[0] = v.x; r[1] = v.y;
    } else {
      r[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < COUNT / 2; ++i) {
      const uint32_t lo = 2 * i < valid ? q[2 * i] : 0, hi = 2 * i + 1 < valid ? q[2 * i + 1] : 0;
      r[i] = lo | hi << 16;
    }
  }
}

// Rows of a chunk by adapter.
template <int ROWS>
struct RowGroupsOf {
  alignas(16) int id[ROWS];
  alignas(16) int leader[ROWS];  // the adapter at its first row, elsewhere a number above all
  int order[ROWS];               // rows of the chunk, those of one adapter together, in their order
  int start[ROWS + 1];           // first place of a group
  int adapter[ROWS];
};
using RowGroups = RowGroupsOf<kChunkRows>;

struct Ids {
  const void* at;  // int32, or int64 with `wide`
  int wide;
};
__device__ __forceinline__ int adapter_of(const Ids& ids, int row, int rows, int L) {  // -1: none
  if (row >= rows) return -1;
  const long long id = ids.wide ? static_cast<const long long*>(ids.at)[row] : (long long)static_cast<const int*>(ids.at)[row];
  return id >= 0 && id < L ? int(id) : -1;
}

// Called by all threads of the CTA, ROWS at least. Returns the number of groups.
template <int ROWS>
__device__ __forceinline__ int group_rows(RowGroupsOf<ROWS>& g, const Ids& ids, int row0, int rows, int L) {
  const int t = threadIdx.x;
  const int first_id = adapter_of(ids, row0, rows, L);
  const int mine = t < ROWS ? adapter_of(ids, row0 + t, rows, L) : first_id;
  if (t < ROWS) g.id[t] = mine;
  if (__syncthreads_and(mine == first_id || (t < ROWS && row0 + t >= rows))) {  // one sequence: the usual chunk of a prefill
    const int count = first_id < 0 ? 0 : min(ROWS, rows - row0);
    if (t < ROWS) g.order[t] = t;
    if (t == 0) {
      g.start[0] = 0;
      g.start[1] = count;
      g.adapter[0] = first_id;
    }
    __syncthreads();
    return count > 0 ? 1 : 0;
  }
  int before = 0;
  bool first = t < ROWS && mine >= 0;
  if (first) {
#pragma unroll
    for (int j = 0; j < ROWS; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(g.id + j);
      const int v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool same_before = v[i] == mine && j + i < t;
        before += (v[i] >= 0 && v[i] < mine) || same_before;
        first &= !same_before;
      }
    }
    g.order[before] = t;
  }
  if (t < ROWS) g.leader[t] = first ? mine : 0x7fffffff;
  const int placed = __syncthreads_count(t < ROWS && mine >= 0);
  const int groups = __syncthreads_count(first);
  if (first) {
    int at = 0;
#pragma unroll
    for (int j = 0; j < ROWS; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(g.leader + j);
      at += (o.x < mine) + (o.y < mine) + (o.z < mine) + (o.w < mine);
    }
    g.start[at] = before;
    g.adapter[at] = mine;
  }
  if (t == 0) g.start[groups] = placed;
  __syncthreads();
  return groups;
}

// The same for a chunk of up to 32 rows, by every warp for itself: the rows of the n-th adapter (in the order of its first row) as a mask, 0 behind the
// last one.
constexpr int kFewRows = 32;
struct FewRows {
  unsigned rows, none;  // of the group; without an adapter
  int adapter;
};
__device__ __forceinline__ FewRows few_rows(const Ids& ids, int row0, int rows, int L, int n) {
  const int lane = threadIdx.x & 31;
  const int mine = adapter_of(ids, row0 + lane, rows, L);
  const unsigned same = __match_any_sync(0xffffffffu, mine);
  const unsigned none = __ballot_sync(0xffffffffu, mine < 0 && row0 + lane < rows);
  const bool first = mine >= 0 && lane == __ffs(same) - 1;
  const unsigned leaders = __ballot_sync(0xffffffffu, first);
  const bool picked = first && __popc(leaders & ((1u << lane) - 1u)) == n;
  const int at = __ffs(__ballot_sync(0xffffffffu, picked)) - 1;
  if (at < 0) return {0u, none, -1};
  return {__shfl_sync(0xffffffffu, same, at), none, __shfl_sync(0xffffffffu, mine, at)};
}
// Place of the n-th bit that is set, -1 behind the last.
__device__ __forceinline__ int nth_bit(unsigned mask, int n) {
  for (int i = 0; i < n; ++i) mask &= mask - 1u;
  return __ffs(mask) - 1;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {  // zeros where not real
  const uint32_t bytes = real ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_bytes(uint32_t dst, const void* src, uint32_t bytes) {  // zeros behind `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Eight bf16 to 16 bytes of shared memory: asynchronously where they may be loaded as one piece, otherwise one by one; zeros behind `valid`.
__device__ __forceinline__ void copy8(uint32_t dst, const __nv_bfloat16* src, const __nv_bfloat16* fallback, bool vec, int valid) {
  if (vec) {
    cp_async16(dst, valid > 0 ? src : fallback, valid > 0);
  } else {
    uint32_t r[4] = {0u, 0u, 0u, 0u};
    if (valid > 0) load_bf16<8>(src, false, valid, r);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
  }
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// Place of 16-byte piece c in a row of PIECES pieces (2, 4, 8 or 16): eight neighbouring rows at one c lie in different banks.
template <int PIECES>
__device__ __forceinline__ uint32_t piece(int row, int c) {
  constexpr int PER_LINE = PIECES >= 8 ? 1 : 8 / PIECES;  // rows to 128 bytes
  return uint32_t((row * PIECES + (c ^ ((row / PER_LINE) & (PIECES >= 8 ? 7 : PIECES - 1)))) * 16);
}

// Two f32 values as three pairs of bf16 that add up to them: a part is the upper half of what the ones before it leave, the next 8 bits of the
// significand, so that no part is rounded. An infinity or NaN is whole in its first part.
constexpr int kParts = 3;
__device__ __forceinline__ float behind_first(float v) {
  const float rest = v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  return fabsf(v) < INFINITY ? rest : 0.f;
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&part)[kParts]) {
  part[0] = high_halves(__float_as_uint(a), __float_as_uint(b));
  const float a1 = behind_first(a), b1 = behind_first(b);
  part[1] = high_halves(__float_as_uint(a1), __float_as_uint(b1));
  const float a2 = a1 - __uint_as_float(__float_as_uint(a1) & 0xffff0000u), b2 = b1 - __uint_as_float(__float_as_uint(b1) & 0xffff0000u);
  part[2] = high_halves(__float_as_uint(a2), __float_as_uint(b2));
}

struct ShrinkParams {
  const __nv_bfloat16* x;  // [rows, K], pitch ldx
  const __nv_bfloat16* w;  // A_l [L][R][K], or (TRANS) B_l [L][K][R]
  Ids ids;
  const float* scale;      // [L], or null
  float* hidden;           // [rows][Rp]
  long long ldx;
  int rows, K, R, Rp, L, split_k;
  int x_vec, w_vec;        // 16-byte loads of x; vector loads of w
};

// A split's sums of `count` rows and COLS ranks are in `sums` ([..][COLS + 1]) of every CTA of the cluster: this CTA adds up its share of the
// rows over the splits, in their order, and writes them, scaled. By its place, a row's: number in `sums`, row of x, scale.
template <int COLS, typename SumRow, typename RowOf, typename ScaleOf>
__device__ __forceinline__ void finish_hidden(const ShrinkParams& p, float* sums, SumRow sum_row, RowOf row_of, ScaleOf scale_of, int count, int n0) {
  __syncthreads();
  const int splits = gridDim.x, split = blockIdx.x;
  if (splits > 1) {
    cluster_arrive();
    cluster_wait();
  }
  const int r0 = count * split / splits, r1 = count * (split + 1) / splits;
  for (int e = threadIdx.x; e < (r1 - r0) * COLS; e += kAdapterThreads) {
    const int row = r0 + e / COLS, col = e % COLS;
    if (n0 + col >= p.Rp) continue;
    float v = 0.f;
    if (splits == 1) {
      v = sums[sum_row(row) * (COLS + 1) + col];
    } else {
      const uint32_t at = smem_u32(sums + sum_row(row) * (COLS + 1) + col);
      float part[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) part[s] = s < splits ? ld_cluster_f32(mapa_shared(at, s)) : 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) v += part[s];
    }
    const int at_row = row_of(row);
    if (WB_CHECK(at_row >= 0 && at_row < p.rows, kCheckOutputIndex, at_row))
      p.hidden[(long long)at_row * p.Rp + n0 + col] = n0 + col < p.R ? v * scale_of(row) : 0.f;  // (an infinity of x would be a NaN in the ranks behind the last)
  }
  if (splits > 1) {  // nobody overwrites what others still read
    cluster_arrive();
    cluster_wait();
  }
  __syncthreads();
}

// hidden[t][r] = scale_l sum_k x[t, k] w_l[r, k]. Grid (splits of K = one cluster, chunks, group lanes).
//
// Few rows: operands straight from global memory to registers. The 8 warps of a CTA take blocks of 64 k in turn. Bound by latency: launch, ids, one
// round of loads, the sum over the warps, the sum over the cluster; one row, K = N = 4096, rank 16: 5.0 us with the expansion behind it.
template <int RT, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_shrink_few_kernel(const ShrinkParams p) {
  constexpr int KU = 2, COLS = RT * 8;
  __shared__ float red[kAdapterWarps][16][COLS + 2];
  __shared__ float sums[16][COLS];  // 16 / splits rows of this CTA from every split (a power of two)
  bool again = false;
  if (gridDim.x > 1) {  // every CTA has begun before the first store into its shared memory; here, where the kernel before this one still runs
    cluster_arrive();
    cluster_wait();
  }
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * kFewRows;
  const int k0 = blockIdx.x * p.split_k, k1 = min(p.K, k0 + p.split_k);
  for (int gi = blockIdx.z;; gi += gridDim.z) {
    const FewRows group = few_rows(p.ids, row0, p.rows, p.L, gi);
    if (group.rows == 0u) break;
    const __nv_bfloat16* w = p.w + (long long)group.adapter * p.R * p.K;
    const float scale = p.scale ? p.scale[group.adapter] : 1.f;
    const int end = __popc(group.rows);
    for (int first = 0; first < end; first += 16) {
      const __nv_bfloat16* src[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = nth_bit(group.rows, first + h * 8 + g);
        src[h] = at >= 0 ? p.x + (long long)(row0 + at) * p.ldx : nullptr;
      }
      for (int n0 = 0; n0 < p.Rp; n0 += COLS) {
        float acc[RT][4] = {};
        for (int kb = k0 + warp * (KU * 32); kb < k1; kb += kAdapterWarps * KU * 32) {
          uint32_t xa[KU][2][4];
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            const int k = kb + u * 32 + t * 8;
            const int valid = min(8, k1 - k);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (src[h] && valid > 0) load_bf16<8>(src[h] + k, p.x_vec != 0, valid, xa[u][h]);
              else xa[u][h][0] = xa[u][h][1] = xa[u][h][2] = xa[u][h][3] = 0u;
            }
          }
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            const int k = kb + u * 32 + t * 8;
            uint32_t wf[RT][4];  // k pairs (0 1) (2 3) (4 5) (6 7) of the lane's eight
            if constexpr (!TRANS) {
              const int valid = min(8, k1 - k);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                const int r = n0 + i * 8 + g;
                if (r < p.R && valid > 0) load_bf16<8>(w + (long long)r * p.K + k, p.w_vec != 0, valid, wf[i]);
                else wf[i][0] = wf[i][1] = wf[i][2] = wf[i][3] = 0u;
              }
            } else {
              uint32_t raw[8][RT / 2];
              const int r = n0 + g * RT;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (k + i < k1 && r < p.R) load_bf16<RT>(w + (long long)(k + i) * p.R + r, p.w_vec != 0 && r + RT <= p.R, p.R - r, raw[i]);
                else
#pragma unroll
                  for (int j = 0; j < RT / 2; ++j) raw[i][j] = 0u;
              }
#pragma unroll
              for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  wf[i][q] = i & 1 ? high_halves(raw[2 * q][i / 2], raw[2 * q + 1][i / 2]) : low_halves(raw[2 * q][i / 2], raw[2 * q + 1][i / 2]);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
              for (int s = 0; s < 2; ++s)
                mma_bf16(acc[i], xa[u][0][2 * s], xa[u][1][2 * s], xa[u][0][2 * s + 1], xa[u][1][2 * s + 1], wf[i][2 * s], wf[i][2 * s + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int col = TRANS ? RT * (2 * t + (c & 1)) + i : i * 8 + 2 * t + (c & 1);
            red[warp][g + (c >> 1) * 8][col] = acc[i][c];
          }
        // every split sends its sums of a row to the CTA that finishes it, which adds them up in their order
        const int count = min(16, end - first), splits = gridDim.x, split = blockIdx.x, share = 16 / splits;
        __syncthreads();
        if (again && splits > 1) {  // what came before has been read
          cluster_arrive();
          cluster_wait();
        }
        again = true;
        for (int e = threadIdx.x; e < count * COLS; e += kAdapterThreads) {
          const int row = e / COLS, col = e % COLS;
          float v = 0.f;
#pragma unroll
          for (int i = 0; i < kAdapterWarps; ++i) v += red[i][row][col];
          const int owner = row % splits;
          float* to = &sums[split * share + row / splits][col];
          if (owner == split) *to = v;
          else asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(to), owner)), "f"(v) : "memory");
        }
        __syncthreads();
        if (splits > 1) {
          cluster_arrive();
          cluster_wait();
        }
        for (int e = threadIdx.x; e < count * COLS; e += kAdapterThreads) {
          const int mine = e / COLS, col = e % COLS, row = mine * splits + split;
          if (row >= count) break;
          if (n0 + col >= p.Rp) continue;
          float v = 0.f;
          for (int i = 0; i < splits; ++i) v += sums[i * share + mine][col];
          const int at_row = row0 + nth_bit(group.rows, first + row);
          if (WB_CHECK(at_row >= row0 && at_row < p.rows, kCheckOutputIndex, at_row)) p.hidden[(long long)at_row * p.Rp + n0 + col] = n0 + col < p.R ? v * scale : 0.f;
        }
      }
    }
  }
}

// Many rows: a ring of stages of 64 k in shared memory, rows of x gathered by their place in the group. Warp (m, q) takes rows 32 m .. and the
// q-th 16 of the 64 k: x passes through ldmatrix once, w twice, and the four sums over k meet at the end. Two stages between barriers, so that the warps
// wait for one another half as often. Bound by HBM on x at rank 16 and by shared memory and issue slots at rank 64, where each 64 rows x 64 k take as
// many ldmatrix of w as of x: 8192 x 8192 at rank 64 48 us (134 MB of x, 2.8 TB/s; MMA pipe 39 %), where the tensor cores take 30 to 33;
// 4096 x 4096 at rank 16 12.7 us.
template <int RT>
struct ShrinkTile {
  static constexpr int X_BYTES = kChunkRows * 128, W_BYTES = RT * 1024, STAGE_BYTES = X_BYTES + W_BYTES;
  static constexpr int STAGES = RT == 8 ? 6 : 8;
  static constexpr int PER_SYNC = 2;  // stages that are worked on between two barriers
  static constexpr int GROUPS = STAGES / PER_SYNC;
  static constexpr int COLS = RT * 8;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES;  // the sums reuse it
  static_assert(STAGES % PER_SYNC == 0 && 4 * kChunkRows * (COLS + 1) * 4 <= SMEM_BYTES, "whole groups; sums of the four k quarters");
};
template <int RT, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_shrink_tile_kernel(const ShrinkParams p) {
  using Cfg = ShrinkTile<RT>;
  constexpr int STAGES = Cfg::STAGES, COLS = Cfg::COLS;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ RowGroups groups;
  const uint32_t base = smem_u32(smem);
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp & 1, wq = warp >> 1;
  const int row0 = blockIdx.y * kChunkRows;
  const int ngroups = group_rows(groups, p.ids, row0, p.rows, p.L);
  const int k0 = blockIdx.x * p.split_k, k1 = min(p.K, k0 + p.split_k);
  const int steps = max(0, (k1 - k0 + 63) / 64);
  for (int gi = blockIdx.z; gi < ngroups; gi += gridDim.z) {
    const int first = groups.start[gi], count = groups.start[gi + 1] - first;
    const int l = groups.adapter[gi];
    const __nv_bfloat16* w = p.w + (long long)l * p.R * p.K;
    const float scale = p.scale ? p.scale[l] : 1.f;
    // A thread brings the same pieces of every stage: of rows tid / 8 and tid / 8 + 32 of x, and WN of w.
    constexpr int WN = (RT * 64 + kAdapterThreads - 1) / kAdapterThreads;
    const int xr = tid >> 3, xc = tid & 7;
    const __nv_bfloat16* row_of_x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) row_of_x[h] = xr + 32 * h < count ? p.x + (long long)(row0 + groups.order[first + xr + 32 * h]) * p.ldx + k0 + xc * 8 : nullptr;
    for (int n0 = 0; n0 < p.Rp; n0 += COLS) {
      // a piece that is not there (a row behind the group's last, a rank behind R) is zeros: its address stays where it is, with a size of 0
      const __nv_bfloat16 *xsrc[2], *wsrc[WN];
      int x_there[2], w_there[WN], w_k[WN];  // elements of a piece that are there; its first k in a stage
      uint32_t xdst[2], wdst[WN];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x_there[h] = row_of_x[h] ? 8 : 0;
        xsrc[h] = row_of_x[h] ? row_of_x[h] : p.x;
        xdst[h] = piece<8>(xr + 32 * h, xc);
      }
#pragma unroll
      for (int i = 0; i < WN; ++i) {
        const int e = tid + i * kAdapterThreads;
        if constexpr (!TRANS) {  // [rank][64 k]
          const int r = e >> 3, c = e & 7;
          w_k[i] = c * 8;
          w_there[i] = e < COLS * 8 && n0 + r < p.R ? 8 : 0;
          wsrc[i] = w_there[i] ? w + (long long)(n0 + r) * p.K + k0 + c * 8 : p.w;
          wdst[i] = Cfg::X_BYTES + piece<8>(r, c);
        } else {  // [k][ranks]
          const int k = e / RT, c = e % RT;
          w_k[i] = k;
          w_there[i] = e < 64 * RT ? max(0, min(8, p.R - n0 - c * 8)) : 0;
          wsrc[i] = w_there[i] ? w + (long long)(k0 + k) * p.R + n0 + c * 8 : p.w;
          wdst[i] = Cfg::X_BYTES + piece<RT>(k, c);
        }
      }
      const bool w_mine = RT * 64 >= kAdapterThreads || tid < RT * 64;
      const long long w_step = TRANS ? 64ll * p.R : 64ll;
      const bool fast = p.x_vec && p.w_vec;
      int left = k1 - k0;        // k that are not loaded yet
      uint32_t to = base;        // first stage of the next load
      constexpr uint32_t LAST = (STAGES - Cfg::PER_SYNC) * Cfg::STAGE_BYTES;
      auto load_group = [&]() {
        if (fast && left >= 64 * Cfg::PER_SYNC) {  // whole pieces
#pragma unroll
          for (int sub = 0; sub < Cfg::PER_SYNC; ++sub) {
#pragma unroll
            for (int h = 0; h < 2; ++h) cp_async_bytes(to + sub * Cfg::STAGE_BYTES + xdst[h], xsrc[h] + (x_there[h] ? sub * 64 : 0), 2 * x_there[h]);
#pragma unroll
            for (int i = 0; i < WN; ++i)
              if (w_mine) cp_async_bytes(to + sub * Cfg::STAGE_BYTES + wdst[i], wsrc[i] + (w_there[i] ? sub * w_step : 0), w_there[i] ? 16 : 0);
          }
        } else {
#pragma unroll
          for (int sub = 0; sub < Cfg::PER_SYNC; ++sub) {
            const int rest = left - 64 * sub;
            if (rest <= 0) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              copy8(to + sub * Cfg::STAGE_BYTES + xdst[h], xsrc[h] + sub * 64, p.x, p.x_vec != 0, x_there[h] ? min(8, rest - xc * 8) : 0);
#pragma unroll
            for (int i = 0; i < WN; ++i)
              if (w_mine)
                copy8(to + sub * Cfg::STAGE_BYTES + wdst[i], wsrc[i] + sub * w_step, p.w, p.w_vec != 0, TRANS ? (w_k[i] < rest ? w_there[i] : 0) : min(w_there[i], rest - w_k[i]));
          }
        }
        cp_async_commit();
        left -= 64 * Cfg::PER_SYNC;
        to = to == base + LAST ? base : to + Cfg::PER_SYNC * Cfg::STAGE_BYTES;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (x_there[h]) xsrc[h] += 64 * Cfg::PER_SYNC;
#pragma unroll
        for (int i = 0; i < WN; ++i)
          if (w_there[i]) wsrc[i] += Cfg::PER_SYNC * w_step;
      };
      const int half = lane >> 4, in = lane & 15;
      const uint32_t xoff = piece<8>(32 * wm + in, 2 * wq + half);  // 16 rows on: 2048 bytes, the same swizzle
      uint32_t woff[RT / 2];
#pragma unroll
      for (int i = 0; i < RT; i += 2)
        woff[i / 2] = Cfg::X_BYTES + (TRANS ? piece<RT>(16 * wq + in, i + half) : piece<8>(half * 8 + (in & 7), 2 * wq + (in >> 3)) + i * 1024);
      uint32_t from = base;
      float acc[2][RT][4] = {};
#pragma unroll
      for (int i = 0; i < Cfg::GROUPS - 1; ++i) load_group();
      for (int step = 0; step < steps; step += Cfg::PER_SYNC) {
        cp_async_wait<Cfg::GROUPS - 2>();
        __syncthreads();
        load_group();
#pragma unroll
        for (int sub = 0; sub < Cfg::PER_SYNC; ++sub) {
          if (32 * wm < count && step + sub < steps) {
            uint32_t xa[2][4];
#pragma unroll
            for (int m = 0; m < 2; ++m) ldsm4(from + xoff + sub * Cfg::STAGE_BYTES + m * 2048, xa[m]);
#pragma unroll
            for (int i = 0; i < RT; i += 2) {
              uint32_t wf[4];
              if constexpr (!TRANS) ldsm4(from + woff[0] + sub * Cfg::STAGE_BYTES + i * 1024, wf);
              else ldsm4_trans(from + woff[i / 2] + sub * Cfg::STAGE_BYTES, wf);
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                mma_bf16(acc[m][i], xa[m][0], xa[m][1], xa[m][2], xa[m][3], wf[0], wf[1]);
                mma_bf16(acc[m][i + 1], xa[m][0], xa[m][1], xa[m][2], xa[m][3], wf[2], wf[3]);
              }
            }
          }
        }
        from = from == base + LAST ? base : from + Cfg::PER_SYNC * Cfg::STAGE_BYTES;
      }
      cp_async_wait<0>();
      __syncthreads();
      float* sums = reinterpret_cast<float*>(smem);  // [4 quarters of k][64][COLS + 1]
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            sums[(wq * kChunkRows + 32 * wm + 16 * m + g + (c >> 1) * 8) * (COLS + 1) + i * 8 + 2 * t + (c & 1)] = acc[m][i][c];
      __syncthreads();
      for (int e = tid; e < count * COLS; e += kAdapterThreads) {
        const int at = e / COLS * (COLS + 1) + e % COLS;
        float v = sums[at];
#pragma unroll
        for (int q = 1; q < 4; ++q) v += sums[q * kChunkRows * (COLS + 1) + at];
        sums[at] = v;
      }
      finish_hidden<COLS>(p, sums, [](int row) { return row; }, [&](int row) { return row0 + groups.order[first + row]; }, [&](int) { return scale; }, count, n0);
    }
  }
}

// The same for many aligned rows and K a multiple of 64, on the tensor cores: the 128 rows of a chunk x N ranks of two adapters at a time, accumulators
// of N columns for each; a row takes the sums of its own. Rows come as one tile, w as one a adapter: A_l's rows K-major, B_l's (TRANS) as they
// lie, with the ranks in an MN-major operand. Ranks behind the last are the next adapter's or zeros and are not kept. No load passes through
// registers, w is read once for 128 rows, and a chunk in which one sequence ends and another begins takes a third longer than others.
// 8192 x 8192 at rank 64 33 us for six sequences, 30 for one (134 MB, 4.1 and 4.5 TB/s). Bound by HBM, which 128 bytes of a row at a time do not bring to its full
// rate; 256 bytes fetched into L2 at a time gained 2 us. Rows gathered by the copy engine, four to a request, took 55.
template <int N, bool TRANS>
struct ShrinkWide {
  static constexpr int ROWS = 128, X_BYTES = ROWS * 128, W_BYTES = TRANS ? 64 * 128 : N * 128, STAGE_BYTES = X_BYTES + 2 * W_BYTES;
  static constexpr int STAGES = STAGE_BYTES > 24 * 1024 ? 3 : 4;
  // Two CTAs to an SM, which share its columns, and beside them none of the library's other kernels that take tensor memory: a CTA holds its columns
  // while it waits for its cluster.
  static constexpr int SMEM_BYTES = 97 * 1024;           // the sums reuse the stages
  // Two accumulators to an adapter, taken in turn by the stages: an MMA drops the bits of its f32 sum that do not fit, always towards zero, and 2048 k in one
  // accumulator shrink by 1.8e-6 of themselves where an f32 sum with rounding is 1e-6 off at random.
  static constexpr int ACCS = 2;
  static constexpr int TMEM_COLS = N < 32 ? 128 : 4 * N;  // (32 columns are read at a time)
  static_assert(STAGES * STAGE_BYTES + 1024 <= SMEM_BYTES && 2 * TMEM_COLS <= 512, "stages; columns of two CTAs");
  static_assert(SMEM_BYTES + kSmemOfTmemKernel > kSmemOfSm && 3 * SMEM_BYTES > kSmemOfSm, "no other kernel with tensor memory beside one CTA, no third CTA");
  static_assert((2 * ACCS - 1) * N + (N < 32 ? 32 : N) <= TMEM_COLS, "accumulators of two adapters");
  static_assert(ROWS * (N + 1) * 4 <= STAGES * STAGE_BYTES && ROWS <= kAdapterThreads, "sums; a thread per row where rows are grouped");
};
template <int N, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_shrink_wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const ShrinkParams p, int* status) {
  using Cfg = ShrinkWide<N, TRANS>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ RowGroupsOf<Cfg::ROWS> groups;
  __shared__ __align__(8) uint64_t bars[2 * Cfg::STAGES + 1];
  __shared__ uint32_t tmem_slot, abort_word;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* sums = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)));  // [128][N + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto full = [&](uint32_t st) { return smem_u32(bars + st); };
  auto empty = [&](uint32_t st) { return smem_u32(bars + Cfg::STAGES + st); };
  const uint32_t acc_full = smem_u32(bars + 2 * Cfg::STAGES);
  WaitCtx ctx{&abort_word, status};
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * Cfg::STAGES + 1; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_word = 0u;
    fence_mbar_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(&tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.y * Cfg::ROWS;
  const int ngroups = group_rows(groups, p.ids, row0, p.rows, p.L);
  const int k0 = blockIdx.x * p.split_k, steps = max(0, min(p.K, k0 + p.split_k) - k0) / 64;  // K and split_k are multiples of 64
  uint32_t stage = 0, phase = 0, acc_phase = 0;
  for (int gi = 2 * blockIdx.z; gi < ngroups; gi += 2 * gridDim.z) {
    const int ng = min(2, ngroups - gi);
    const int first = groups.start[gi], middle = groups.start[gi + 1], count = groups.start[gi + ng] - first;
    const int l[2] = {groups.adapter[gi], groups.adapter[gi + ng - 1]};
    const float scale[2] = {p.scale ? p.scale[l[0]] : 1.f, p.scale ? p.scale[l[1]] : 1.f};
    for (int n0 = 0; n0 < p.Rp; n0 += N) {
      if (warp == 0) {
        for (int s = 0; s < steps; ++s) {
          if (!mbar_wait(empty(stage), phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;  // given up: nothing more is issued
          const uint32_t to = base + stage * Cfg::STAGE_BYTES;
          const int k = k0 + s * 64;
          if (elect_one()) {
            mbar_expect_tx(full(stage), uint32_t(Cfg::X_BYTES + ng * Cfg::W_BYTES));
            tma_load_2d<1>(to, &map_x, k, row0, full(stage));
            for (int i = 0; i < ng; ++i) {
              if constexpr (TRANS) tma_load_2d<1>(to + Cfg::X_BYTES + i * Cfg::W_BYTES, &map_w, n0, l[i] * p.K + k, full(stage));
              else tma_load_2d<1>(to + Cfg::X_BYTES + i * Cfg::W_BYTES, &map_w, k, l[i] * p.R + n0, full(stage));
            }
          }
          __syncwarp();
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1u; }
        }
      } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc_bf16_bt(Cfg::ROWS, N) & ~(TRANS ? 0u : 1u << 16);  // B K-major, or MN-major
        for (int s = 0; s < steps; ++s) {
          mbar_wait(full(stage), phase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
          tc_fence_after_sync();
          const uint32_t at = base + stage * Cfg::STAGE_BYTES;
          if (elect_one()) {
            const uint64_t a = make_desc_k_sw128(at);
            for (int i = 0; i < ng; ++i) {
              const uint32_t w_at = at + Cfg::X_BYTES + i * Cfg::W_BYTES;
              const uint64_t b = TRANS ? make_desc_mn_sw128(w_at, 64 * 128) : make_desc_k_sw128(w_at);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16<1>(tmem + (i * Cfg::ACCS + s % Cfg::ACCS) * N, a + uint64_t(k * 2), b + uint64_t(k * (TRANS ? 2048 >> 4 : 2)), idesc,
                           (s >= Cfg::ACCS || k > 0) ? 1u : 0u);
            }
            tc_commit<1>(empty(stage));
            if (s == steps - 1) tc_commit<1>(acc_full);
          }
          __syncwarp();
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (steps > 0) {
        mbar_wait(acc_full, acc_phase, ctx, WB_DEV_TIMEOUT_EPILOGUE);
        acc_phase ^= 1u;
        tc_fence_after_sync();
      }
      // warps w and w + 4 read rows 32 (w % 4) .., 32 columns each; every stage has been read by now
      const int row = (warp & 3) * 32 + lane, c = (warp >> 2) * 32;
      if (c < N) {
        for (int i = 0; i < ng; ++i) {
          float sum[32] = {};
          for (int a = 0; a < min(steps, Cfg::ACCS); ++a) {
            uint32_t v[32];
            tmem_ld_32x32(tmem + (uint32_t((warp & 3) * 32) << 16) + (i * Cfg::ACCS + a) * N + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[j] += __uint_as_float(v[j]);
          }
          if (groups.id[row] == l[i])
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < N) sums[row * (N + 1) + c + j] = sum[j];
        }
      }
      tc_fence_before_sync();
      finish_hidden<N>(
          p, sums, [&](int place) { return groups.order[first + place]; }, [&](int place) { return row0 + groups.order[first + place]; },
          [&](int place) { return first + place < middle ? scale[0] : scale[1]; }, count, n0);
      fence_proxy_async_smem();  // the copy engine writes next where the sums have been read
      __syncthreads();
      tc_fence_after_sync();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
  }
}

struct ExpandParams {
  const __nv_bfloat16* w;       // B_l [L][C][R], or (TRANS) A_l [L][R][C]
  Ids ids;
  const float* hidden;          // [rows][Rp]
  const void* y;                // null: zeros
  void* out;
  long long ldy, ldo;
  int rows, C, R, Rp, L, cols_per_cta;
  int io_vec, w_vec, io_pairs;  // rows of y and out start on 16 bytes; vector loads of w; bf16 rows start on 4 bytes and C is even
};

template <typename T>
__device__ __forceinline__ float as_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T as_out(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ void read8(const T* p, bool whole, int valid, float (&v)[8]) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r[i] << 16); v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? as_f32<T>(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void write8(T* p, bool whole, int valid, const float (&v)[8]) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = as_out<T>(v[i]);
  }
}


// A row without an adapter: y as it is (zeros where there is no y).
template <typename T>
__device__ __forceinline__ void expand_rest(const ExpandParams& p, long long row, int c, int c_end, int step) {
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  for (; c < c_end; c += step) {
    const int valid = c_end - c;
    float v[8] = {};
    if (y) read8<T>(y + row * p.ldy + c, p.io_vec && valid >= 8, valid, v);
    if (WB_CHECK(row < p.rows && c < p.C && c_end <= p.C, kCheckOutputIndex, row << 32 | c)) write8<T>(out + row * p.ldo + c, p.io_vec && valid >= 8, valid, v);
  }
}

// out[t, c] = y[t, c] + sum_r hidden[t, r] w_l[c, r]. Grid (column slices, chunks, group lanes).
//
// Few rows: a thread has two columns, with 16 of their ranks in registers at a time, and walks the rows of a group. f32 FMAs: the
// products are few, the loads of w_l (whole sectors, all of a thread's in flight) are what counts. For ranks and alignments that the next kernel does not
// take, and for the transposed product of the backward pass.
template <typename T, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_expand_few_kernel(const ExpandParams p) {
  constexpr int ROWS = 8;
  extern __shared__ __align__(16) float hs[];  // [ROWS][Rp]
  pdl_launch_dependents();
  const int row0 = blockIdx.y * kFewRows;
  const int c_begin = blockIdx.x * p.cols_per_cta, c_end = min(p.C, c_begin + p.cols_per_cta);
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const int c = c_begin + 2 * threadIdx.x;  // cols_per_cta is twice the number of threads
  const bool both = c + 1 < c_end;
  bool waited = false;
  unsigned none = 0u;
  for (int gi = blockIdx.z;; gi += gridDim.z) {
    const FewRows group = few_rows(p.ids, row0, p.rows, p.L, gi);
    none = group.none;
    if (group.rows == 0u) break;
    const __nv_bfloat16* w = p.w + (long long)group.adapter * p.R * p.C;
    unsigned rest = group.rows;
    while (rest != 0u) {
      int row[ROWS];
      int count = 0;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        row[i] = row0 + __ffs(rest) - 1;
        count += rest != 0u;
        rest &= rest - 1u;
      }
      float acc[ROWS][2];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        acc[i][0] = acc[i][1] = 0.f;
        if (y && i < count && c < c_end) {
          const T* at = y + row[i] * p.ldy + c;
          if (p.io_vec && both) {
            if constexpr (sizeof(T) == 2) {
              const uint32_t v = *reinterpret_cast<const uint32_t*>(at);
              acc[i][0] = __uint_as_float(v << 16);
              acc[i][1] = __uint_as_float(v & 0xffff0000u);
            } else {
              const float2 v = *reinterpret_cast<const float2*>(at);
              acc[i][0] = v.x;
              acc[i][1] = v.y;
            }
          } else {
            acc[i][0] = as_f32<T>(at[0]);
            if (both) acc[i][1] = as_f32<T>(at[1]);
          }
        }
      }
      for (int r0 = 0; r0 < p.Rp; r0 += 16) {
        uint32_t wr[2][8];  // column, pairs of ranks
        if constexpr (!TRANS) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = r0 + 8 * h;
              uint32_t v[4] = {0u, 0u, 0u, 0u};
              if (c + j < c_end && r < p.R) load_bf16<8>(w + (long long)(c + j) * p.R + r, p.w_vec != 0, p.R - r, v);
#pragma unroll
              for (int i = 0; i < 4; ++i) wr[j][4 * h + i] = v[i];
            }
        } else {
          uint32_t raw[16];  // both columns of a rank
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            uint32_t v[1] = {0u};
            if (c < c_end && r0 + i < p.R) load_bf16<2>(w + (long long)(r0 + i) * p.C + c, p.w_vec != 0, both ? 2 : 1, v);
            raw[i] = v[0];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            wr[0][i] = low_halves(raw[2 * i], raw[2 * i + 1]);
            wr[1][i] = high_halves(raw[2 * i], raw[2 * i + 1]);
          }
        }
        if (r0 == 0) {
          if (!waited) pdl_wait();  // the hidden vectors are the only thing here that the kernel before this one writes
          waited = true;
          __syncthreads();
          for (int e = threadIdx.x; e < count * p.Rp; e += kAdapterThreads) {
            const int in = e / p.Rp, r = e - in * p.Rp;
            int from = row[0];
#pragma unroll
            for (int i = 1; i < ROWS; ++i) from = in == i ? row[i] : from;
            hs[e] = p.hidden[(long long)from * p.Rp + r];
          }
          __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          if (i >= count) break;
          const float4* h = reinterpret_cast<const float4*>(hs + i * p.Rp + r0);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 v = h[q];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t a = wr[j][2 * q], b = wr[j][2 * q + 1];
              acc[i][j] = fmaf(v.x, __uint_as_float(a << 16), acc[i][j]);
              acc[i][j] = fmaf(v.y, __uint_as_float(a & 0xffff0000u), acc[i][j]);
              acc[i][j] = fmaf(v.z, __uint_as_float(b << 16), acc[i][j]);
              acc[i][j] = fmaf(v.w, __uint_as_float(b & 0xffff0000u), acc[i][j]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (i >= count || c >= c_end) break;
        if (!WB_CHECK(row[i] >= row0 && row[i] < p.rows && c + int(both) < p.C, kCheckOutputIndex, (long long)row[i] << 32 | c)) continue;
        T* at = out + row[i] * p.ldo + c;
        if (p.io_vec && both) {
          if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(acc[i][0], acc[i][1]);
          else *reinterpret_cast<float2*>(at) = make_float2(acc[i][0], acc[i][1]);
        } else {
          at[0] = as_out<T>(acc[i][0]);
          if (both) at[1] = as_out<T>(acc[i][1]);
        }
      }
    }
  }
  if (!waited) pdl_wait();  // (out may still be in use)
  if (blockIdx.z == 0 && p.out != p.y)
    for (; none != 0u; none &= none - 1u) expand_rest<T>(p, row0 + __ffs(none) - 1, c_begin + threadIdx.x * 8, c_end, kAdapterThreads * 8);
}

// The same for ranks of 8 PIECES whose rows of B start on 16 bytes: PIECES lanes share a column, each with 8 of its ranks, so that a warp's load is 512
// consecutive bytes, STEPS of them in flight; the lanes' sums meet by shuffles, and the u-th lane of a column keeps every so-manieth column.
// Both products of 32 rows and some 25 of 64 adapters, K = 4096, N = 14336, rank 16: 11.8 us (17 MB; with two columns a thread 13.7), of one row
// with N = 4096 5.0 us (6.0).
__host__ __device__ constexpr int few_whole_steps(int pieces) { return pieces > 4 ? pieces : 4; }
template <typename T, int PIECES>
__global__ void __launch_bounds__(kAdapterThreads, 3)
adapter_expand_few_whole_kernel(const ExpandParams p) {
  constexpr int STEPS = few_whole_steps(PIECES), ROWS = 2, KEPT = STEPS / PIECES, COLS = kAdapterThreads / PIECES;  // COLS: of a step
  pdl_launch_dependents();
  const int row0 = blockIdx.y * kFewRows;
  const int c_begin = blockIdx.x * p.cols_per_cta, c_end = min(p.C, c_begin + p.cols_per_cta);  // cols_per_cta = STEPS * COLS
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const int pc = threadIdx.x % PIECES, c = c_begin + threadIdx.x / PIECES;
  bool waited = false;
  unsigned none = 0u;
  for (int gi = blockIdx.z;; gi += gridDim.z) {
    const FewRows group = few_rows(p.ids, row0, p.rows, p.L, gi);
    none = group.none;
    if (group.rows == 0u) break;
    const __nv_bfloat16* w = p.w + (long long)group.adapter * p.R * p.C + pc * 8;
    uint4 wr[STEPS];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) wr[u] = c + u * COLS < c_end ? *reinterpret_cast<const uint4*>(w + (long long)(c + u * COLS) * p.R) : make_uint4(0u, 0u, 0u, 0u);
    unsigned rest = group.rows;
    while (rest != 0u) {
      int row[ROWS], count = 0;
      float old[ROWS][KEPT];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        row[i] = row0 + __ffs(rest) - 1;
        count += rest != 0u;
        rest &= rest - 1u;
#pragma unroll
        for (int k = 0; k < KEPT; ++k) {
          const int col = c + (k * PIECES + pc) * COLS;
          old[i][k] = y && i < count && col < c_end ? as_f32<T>(y[row[i] * p.ldy + col]) : 0.f;
        }
      }
      if (!waited) pdl_wait();  // the hidden vectors are the only thing here that the kernel before this one writes
      waited = true;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (i >= count) break;
        float h[8];
        read8<float>(p.hidden + (long long)row[i] * p.Rp + pc * 8, true, 8, h);
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          float v[8], sum = 0.f;
          read8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(&wr[u]), true, 8, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum = fmaf(h[j], v[j], sum);
#pragma unroll
          for (int o = 1; o < PIECES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (u % PIECES == pc) old[i][u / PIECES] += sum;
        }
#pragma unroll
        for (int k = 0; k < KEPT; ++k) {
          const int col = c + (k * PIECES + pc) * COLS;
          if (col < c_end && WB_CHECK(row[i] >= row0 && row[i] < p.rows && col < p.C, kCheckOutputIndex, (long long)row[i] << 32 | col))
            out[row[i] * p.ldo + col] = as_out<T>(old[i][k]);
        }
      }
    }
  }
  if (!waited) pdl_wait();  // (out may still be in use)
  if (blockIdx.z == 0 && p.out != p.y)
    for (; none != 0u; none &= none - 1u) expand_rest<T>(p, row0 + __ffs(none) - 1, c_begin + threadIdx.x * 8, c_end, kAdapterThreads * 8);
}

// Elements between the hidden vectors of rows in shared memory: a distance at which the loads that move together fall into different banks, those of
// four rows of 8-byte pieces, or (PAIRED) of two rows of 16-byte pieces.
__host__ __device__ constexpr int expand_pitch(int Rp, bool paired) {
  const int words = kParts * Rp / 2;
  return paired ? 2 * (words + (words % 32 == 16 ? 0 : 16)) : 2 * (words + (words % 16 == 8 ? 0 : 8));
}

// Batches of y that are on their way to shared memory at a time: 64 KB of a CTA, 32 KB next to the hidden vectors of ranks that may be large.
__host__ __device__ constexpr int expand_depth(int esz, bool exact) { return (exact ? 8 : 4) / esz; }
__host__ __device__ constexpr int expand_ring_bytes(int esz, bool exact) { return expand_depth(esz, exact) * 2 * esz * kAdapterThreads * 16; }

// Many rows: a warp takes 32 columns of all the rows of a group; a lane has 8 neighbouring columns of two rows of an MMA tile.
// FAST: rows that start on 16 bytes, columns in eights, ranks in fours (eights where two steps are loaded as one piece). The values of y are loaded
// ahead of everything else, a batch of rows (MB tiles of 16) at once, the next batch while this one is worked on, w of the next columns with it;
// they are the accumulators' first values. Otherwise the accumulators go through shared memory, so that 32 lanes share a row's 32 columns, and y a
// row of 32 columns at a time, a tile of 16 rows ahead.
// QN: steps of 16 ranks of w in registers at a time. EXACT: the rank is known when compiled.
// Bound by its start-up and HBM at rank 16 (4096 x 4096 18 us); at rank 64 by the MMA pipe and shared memory between them, at two CTAs of 128 registers a
// thread: 8192 x 8192 97 us (268 MB of y and out, 2.8 TB/s), where the tensor cores take 57 to 61. With the batch ahead in registers instead of the
// ring a fifth slower; w of the next columns through the ring too: no faster.
template <typename T, int QN, bool TRANS, bool FAST, bool EXACT>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_expand_tile_kernel(const ExpandParams p) {
  const int Rp = EXACT ? 16 * QN : p.Rp;         // EXACT: known when compiled, and with it every address in shared memory
  constexpr int RAW = sizeof(T) == 2 ? 1 : 2;    // 16-byte pieces of 8 values
  constexpr int MB = 2;                          // tiles of 16 rows in a batch
  constexpr bool AHEAD = FAST && EXACT && QN <= 2;  // all ranks of w are in registers at a time
  constexpr int STEP = kAdapterWarps * kExpandCols;
  constexpr int DEPTH = expand_depth(sizeof(T), EXACT), SLOT = MB * 2 * RAW * kAdapterThreads * 16;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ RowGroups groups;
  __shared__ uint32_t y_off[FAST ? 1 : kChunkRows], out_off[FAST ? 1 : kChunkRows];  // of a group's rows, in bytes; all ones: none
  __shared__ float staged[FAST ? 1 : kAdapterWarps][FAST ? 1 : 16][FAST ? 1 : kExpandCols + 1];
  // FAST: a ring of batches of y, in which every thread has 16-byte slots of its own (no barrier): [DEPTH][MB][2][RAW][threads]
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(smem + (FAST ? DEPTH * SLOT : 0));  // [64][kParts][Rp], rows `pitch` apart
  // A lane's ranks in two steps of 16: eight neighbours (PAIRED: one 16-byte piece serves both steps), or four of each
  constexpr bool PAIRED = FAST && EXACT && QN % 2 == 0;
  const int pitch = expand_pitch(Rp, PAIRED);
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * kChunkRows;
  const int ngroups = group_rows(groups, p.ids, row0, p.rows, p.L);
  const int c_begin = blockIdx.x * p.cols_per_cta, c_end = min(p.C, c_begin + p.cols_per_cta);
  const int steps = Rp / 16;
  // rows of the chunk, by 32-bit offsets (a pitch is below 2^24 elements)
  const char* y = static_cast<const char*>(p.y) + row0 * p.ldy * int(sizeof(T));
  char* out = static_cast<char*>(p.out) + row0 * p.ldo * int(sizeof(T));
  const uint32_t y_pitch = uint32_t(p.ldy) * sizeof(T), out_pitch = uint32_t(p.ldo) * sizeof(T);
  bool waited = false;
  for (int gi = blockIdx.z; gi < ngroups; gi += gridDim.z) {
    const int first = groups.start[gi], count = groups.start[gi + 1] - first;
    const __nv_bfloat16* w = p.w + (long long)groups.adapter[gi] * p.R * p.C;
    const int mtiles = (count + 15) >> 4;
    auto row_at = [&](int place) { return place < count ? groups.order[first + place] : -1; };
    if constexpr (!FAST) {
      __syncthreads();
      if (threadIdx.x < kChunkRows) {
        const int r = row_at(threadIdx.x);
        y_off[threadIdx.x] = r >= 0 && p.y ? uint32_t(r) * y_pitch : 0xffffffffu;
        out_off[threadIdx.x] = r >= 0 ? uint32_t(r) * out_pitch : 0xffffffffu;
      }
      __syncthreads();
    }
    int row[4][2];  // in the chunk; -1: none
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) row[m][h] = row_at(m * 16 + h * 8 + g);
    const bool has_y = !TRANS || p.y;  // (only a gradient may have nothing to be added to)
    // The next batch of y into the ring: 8 values of every row of it, zeros for a row or column that is not there.
    const uint32_t ring = smem_u32(smem) + threadIdx.x * 16u;
    const int batches = (mtiles + MB - 1) / MB;
    int ahead_c = c_begin + warp * kExpandCols + 8 * t, ahead_batch = 0;
    uint32_t ahead_slot = 0;
    auto load_y = [&]() {
      if (has_y && ahead_c - 8 * t < c_end) {
        const bool col_there = ahead_c < p.C;  // (C is a multiple of 8)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            int r = row[m][h];
#pragma unroll
            for (int b = 1; b < 4 / MB; ++b)
              if (b == ahead_batch) r = row[b * MB + m][h];
            const bool there = col_there && r >= 0;
            const char* from = there ? y + (uint32_t(r) * y_pitch + uint32_t(ahead_c) * uint32_t(sizeof(T))) : reinterpret_cast<const char*>(p.hidden);
#pragma unroll
            for (int i = 0; i < RAW; ++i)
              cp_async_bytes(ring + ahead_slot * SLOT + ((m * 2 + h) * RAW + i) * (kAdapterThreads * 16), from + (there ? 16 * i : 0), there ? 16u : 0u);
          }
        if (++ahead_batch == batches) { ahead_batch = 0; ahead_c += STEP; }
        ahead_slot = ahead_slot + 1 == DEPTH ? 0 : ahead_slot + 1;
      }
      cp_async_commit();
    };
    uint32_t slot = 0;
    uint32_t wf[4][QN][2];
    auto load_w = [&](int c0, int q0) {
      if constexpr (FAST) {
        const int lane_rank = q0 * 16 + (PAIRED ? 8 : 4) * t;
        const int cw = TRANS ? (c0 + 4 * g < p.C ? c0 + 4 * g : 0) : (c0 + 8 * (g >> 1) < p.C ? c0 + 8 * (g >> 1) : 0) + (g & 1);  // (columns as in load_y)
        const __nv_bfloat16* at = TRANS ? w + (long long)lane_rank * p.C + cw : w + (long long)cw * p.R + lane_rank;
#pragma unroll
        for (int q = 0; q < QN; ++q) {
          if (!EXACT && (q0 + q) * 16 >= Rp) break;
          // ranks behind the last are zeros (a lane's piece is there or not: R is a multiple of its ranks)
          const bool rank_there = p.R == Rp || lane_rank + (PAIRED ? q / 2 * 32 : q * 16) < p.R;
          if constexpr (!TRANS && PAIRED) {
            if (q % 2 == 0)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (rank_there) v = *reinterpret_cast<const uint4*>(at + i * (2 * p.R) + q * 16);
                wf[i][q][0] = v.x;
                wf[i][q][1] = v.y;
                wf[i][q + 1 < QN ? q + 1 : q][0] = v.z;
                wf[i][q + 1 < QN ? q + 1 : q][1] = v.w;
              }
          } else if constexpr (!TRANS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint2 v = make_uint2(0u, 0u);
              if (rank_there) v = *reinterpret_cast<const uint2*>(at + i * (2 * p.R) + q * 16);
              wf[i][q][0] = v.x;
              wf[i][q][1] = v.y;
            }
          } else {
            uint2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = PAIRED ? (q / 2) * 32 + (q % 2) * 4 + i : q * 16 + i;
              v[i] = make_uint2(0u, 0u);
              if (p.R == Rp || lane_rank + r < p.R) v[i] = *reinterpret_cast<const uint2*>(at + (long long)r * p.C);
            }
            wf[0][q][0] = low_halves(v[0].x, v[1].x); wf[0][q][1] = low_halves(v[2].x, v[3].x);
            wf[1][q][0] = high_halves(v[0].x, v[1].x); wf[1][q][1] = high_halves(v[2].x, v[3].x);
            wf[2][q][0] = low_halves(v[0].y, v[1].y); wf[2][q][1] = low_halves(v[2].y, v[3].y);
            wf[3][q][0] = high_halves(v[0].y, v[1].y); wf[3][q][1] = high_halves(v[2].y, v[3].y);
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < QN; ++q) {
          const int r = (q0 + q) * 16 + 4 * t;
          uint32_t raw[4][2];
          if constexpr (!TRANS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = c0 + 8 * (g >> 1) + 2 * i + (g & 1);
              if (c < p.C && r < p.R) load_bf16<4>(w + (long long)c * p.R + r, p.w_vec != 0 && r + 4 <= p.R, p.R - r, raw[i]);
              else raw[i][0] = raw[i][1] = 0u;
              wf[i][q][0] = raw[i][0];
              wf[i][q][1] = raw[i][1];
            }
          } else {
            const int c = c0 + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (c < p.C && r + i < p.R) load_bf16<4>(w + (long long)(r + i) * p.C + c, p.w_vec != 0 && c + 4 <= p.C, p.C - c, raw[i]);
              else raw[i][0] = raw[i][1] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                wf[i][q][h] = i & 1 ? high_halves(raw[2 * h][i / 2], raw[2 * h + 1][i / 2]) : low_halves(raw[2 * h][i / 2], raw[2 * h + 1][i / 2]);
          }
        }
      }
    };
    const int c_first = c_begin + warp * kExpandCols;
    // not FAST: a row's 32 columns to the lanes, the rows of a tile at once, those of the next tile ahead
    float old[FAST ? 1 : 16];
    // (bf16 rows that start on 4 bytes: two columns to a lane, two rows to a load)
    const bool pairs = sizeof(T) == 2 && p.io_pairs;
    const int lane_row = pairs ? lane >> 4 : 0, lane_col = pairs ? (lane & 15) * 2 : lane;
    auto load_tile = [&](int c0, int m) {
      const bool there = c0 + lane_col < c_end;
      const uint32_t at = uint32_t(c0 + lane_col) * uint32_t(sizeof(T));
      if (pairs) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t off = y_off[FAST ? 0 : m * 16 + 2 * r + lane_row];
          const uint32_t v = there && off != 0xffffffffu ? *reinterpret_cast<const uint32_t*>(y + (off + at)) : 0u;
          old[FAST ? 0 : 2 * r] = __uint_as_float(v << 16);
          old[FAST ? 0 : 2 * r + 1] = __uint_as_float(v & 0xffff0000u);
        }
        return;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t off = y_off[FAST ? 0 : m * 16 + r];
        old[FAST ? 0 : r] = there && off != 0xffffffffu ? as_f32<T>(*reinterpret_cast<const T*>(y + (off + at))) : 0.f;
      }
    };
    if constexpr (FAST)
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) load_y();
    if (c_first < c_end) {
      if constexpr (!FAST) load_tile(c_first, 0);
      if (AHEAD || (!FAST && steps <= QN)) load_w(c_first, 0);
    }
    if (!waited) pdl_wait();  // for the hidden vectors; y and w are complete before the kernel that makes those starts
    waited = true;
    __syncthreads();
    const int quads = Rp / 4;  // four ranks of a row at a time, the loads of four such pieces in flight
    for (int e0 = threadIdx.x; e0 < mtiles * 16 * quads; e0 += 4 * kAdapterThreads) {
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kAdapterThreads, r = e / quads;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < count) v[i] = *reinterpret_cast<const float4*>(p.hidden + (long long)(row0 + groups.order[first + r]) * Rp + (e - r * quads) * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kAdapterThreads, r = e / quads;
        if (r >= mtiles * 16) break;
        uint32_t lo[kParts], hi[kParts];
        split_pair(v[i].x, v[i].y, lo);
        split_pair(v[i].z, v[i].w, hi);
#pragma unroll
        for (int q = 0; q < kParts; ++q) *reinterpret_cast<uint2*>(hs + r * pitch + q * Rp + (e - r * quads) * 4) = make_uint2(lo[q], hi[q]);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int c0 = c_first; c0 < c_end; c0 += STEP) {
      if (!AHEAD && (FAST || steps > QN || c0 > c_first)) load_w(c0, 0);
      uint32_t wn[4][QN][2];
      if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int q = 0; q < QN; ++q) { wn[i][q][0] = wf[i][q][0]; wn[i][q][1] = wf[i][q][1]; }
        if (c0 + STEP < c_end) load_w(c0 + STEP, 0);
      }
      auto& wu = AHEAD ? wn : wf;
#pragma unroll
      for (int batch = 0; batch < 4 / MB; ++batch) {
        if (batch * MB >= mtiles) break;
        float acc[MB][4][4];
        if constexpr (FAST) cp_async_wait<DEPTH - 1>();
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[8] = {};
            if (FAST && has_y) {
              uint4 raw[RAW];
#pragma unroll
              for (int i = 0; i < RAW; ++i) raw[i] = *reinterpret_cast<const uint4*>(smem + slot * SLOT + ((m * 2 + h) * RAW + i) * (kAdapterThreads * 16) + threadIdx.x * 16);
              read8<T>(reinterpret_cast<const T*>(raw), true, 8, v);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) acc[m][n][2 * h + j] = v[TRANS ? 4 * j + n : 2 * n + j];
          }
        if constexpr (FAST) {
          load_y();
          slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
#pragma unroll
        for (int mm = 0; mm < MB; ++mm) {
          const int m = batch * MB + mm;
          if (m >= mtiles) break;
          for (int q0 = 0; q0 < steps; q0 += QN) {
            if (steps > QN && (q0 > 0 || m > 0)) load_w(c0, q0);
            if constexpr (PAIRED) {
#pragma unroll
              for (int q = 0; q < QN; q += 2) {
                const __nv_bfloat16* at = hs + (m * 16 + g) * pitch + q * 16 + 8 * t;
#pragma unroll
                for (int i = 0; i < kParts; ++i) {
                  const uint4 lo = *reinterpret_cast<const uint4*>(at + i * Rp);
                  const uint4 hi = *reinterpret_cast<const uint4*>(at + 8 * pitch + i * Rp);
#pragma unroll
                  for (int n = 0; n < 4; ++n) mma_bf16(acc[mm][n], lo.x, hi.x, lo.y, hi.y, wu[n][q][0], wu[n][q][1]);
#pragma unroll
                  for (int n = 0; n < 4; ++n) mma_bf16(acc[mm][n], lo.z, hi.z, lo.w, hi.w, wu[n][q + 1][0], wu[n][q + 1][1]);
                }
              }
              break;
            }
#pragma unroll
            for (int q = 0; q < QN; ++q) {
              if (q0 + q >= steps) break;
              const __nv_bfloat16* at = hs + (m * 16 + g) * pitch + (q0 + q) * 16 + 4 * t;
#pragma unroll
              for (int i = 0; i < kParts; ++i) {
                const uint2 lo = *reinterpret_cast<const uint2*>(at + i * Rp);
                const uint2 hi = *reinterpret_cast<const uint2*>(at + 8 * pitch + i * Rp);
#pragma unroll
                for (int n = 0; n < 4; ++n) mma_bf16(acc[mm][n], lo.x, hi.x, lo.y, hi.y, wu[n][q][0], wu[n][q][1]);
              }
            }
          }
          if constexpr (FAST) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (row[m][h] < 0 || c0 + 8 * t >= p.C) continue;
              if (!WB_CHECK(row0 + row[m][h] < p.rows && c0 + 8 * t + 8 <= p.C, kCheckOutputIndex, (long long)(row0 + row[m][h]) << 32 | (c0 + 8 * t))) continue;
              float v[8];
#pragma unroll
              for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) v[TRANS ? 4 * j + n : 2 * n + j] = acc[mm][n][2 * h + j];
              write8<T>(reinterpret_cast<T*>(out + (uint32_t(row[m][h]) * out_pitch + uint32_t(c0 + 8 * t) * uint32_t(sizeof(T)))), true, 8, v);
            }
          } else {
            float (*mine)[kExpandCols + 1] = staged[warp];
            __syncwarp();
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) mine[g + (e >> 1) * 8][8 * t + (TRANS ? 4 * (e & 1) + n : 2 * n + (e & 1))] = acc[mm][n][e];
            __syncwarp();
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = old[FAST ? 0 : r] + (pairs ? mine[(r & ~1) + lane_row][lane_col + (r & 1)] : mine[r][lane]);
            if (m + 1 < mtiles) load_tile(c0, m + 1);
            else if (c0 + STEP < c_end) load_tile(c0 + STEP, 0);
            if (c0 + lane_col < c_end) {
              const uint32_t at = uint32_t(c0 + lane_col) * uint32_t(sizeof(T));
              if (pairs) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                  const uint32_t off = out_off[FAST ? 0 : m * 16 + 2 * r + lane_row];
                  if (off != 0xffffffffu && WB_CHECK(row0 + int(off / out_pitch) < p.rows && c0 + lane_col + 2 <= p.C, kCheckOutputIndex, off))
                    *reinterpret_cast<uint32_t*>(out + (off + at)) = pack_bf16x2(v[2 * r], v[2 * r + 1]);
                }
              } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const uint32_t off = out_off[FAST ? 0 : m * 16 + r];
                  if (off != 0xffffffffu && WB_CHECK(row0 + int(off / out_pitch) < p.rows && c0 + lane_col < p.C, kCheckOutputIndex, off))
                    *reinterpret_cast<T*>(out + (off + at)) = as_out<T>(v[r]);
                }
              }
            }
          }
        }
      }
    }
  }
  if (!waited) pdl_wait();
  if (blockIdx.z == 0 && p.out != p.y)
    for (int r = warp; r < min(kChunkRows, p.rows - row0); r += kAdapterWarps)
      if (groups.id[r] < 0) expand_rest<T>(p, row0 + r, c_begin + lane * 8, c_end, 256);
}

// The same for many aligned bf16 rows and ranks up to 64, on the tensor cores: 128 rows of a chunk x 128 columns, the three parts of the hidden vectors against
// the same tile of w (A operand: the chunk's hidden vectors, split into parts once, by the warps that later read the sums; B: B_l's rows K-major, or
// (TRANS) A_l's as they lie, MN-major). Two adapters at a time have accumulators, a row takes the sums of its own; y comes by the copy engine, is added to in shared memory and leaves from there.
// One CTA per SM works through its share of all (chunk, 128 columns) in order. 8192 x 8192 at rank 64 57 us for one sequence (268 MB, 4.7 TB/s), 61 for six, of
// which 3 are the third part and 3 the loads of the hidden vectors at the head of a chunk; the mma.sync form 97. Bound by HBM, and below 8192 x 4096
// by the start-up of one large CTA per SM.
//   warp 0: y and w by TMA; warp 1: tcgen05.mma; warps 2 .. 9: hidden vectors, then sums, thread = row, 64 columns; warp 10: out by TMA
template <bool TRANS>
struct ExpandWide {
  static constexpr int ROWS = 128, COLS = 128, A_BYTES = kParts * ROWS * 128, B_BYTES = COLS * 128, Y_BYTES = ROWS * COLS * 2;
  static constexpr int B_STAGES = 4, Y_STAGES = 3, EPILOGUE_WARPS = 8, THREADS = (3 + EPILOGUE_WARPS) * 32;
  static constexpr int B_BASE = A_BYTES, Y_BASE = B_BASE + B_STAGES * B_BYTES;
  static constexpr int SMEM_BYTES = Y_BASE + Y_STAGES * Y_BYTES + 1024;
  static constexpr int TMEM_COLS = 512;  // two buffers of two adapters
  static_assert(SMEM_BYTES >= kSmemOfTmemKernel, "keeps other kernels with tensor memory off the SM");
  static_assert(EPILOGUE_WARPS * 32 == 2 * ROWS, "two threads split a row's hidden vector");
};
struct ExpandWideParams {
  Ids ids;
  const float* hidden;  // [rows][Rp]
  int rows, C, R, Rp, L, chunks, tiles;
  int has_y, in_place;
  int* status;
};
// A CTA's share of the tiles. A tile of a chunk in which one sequence ends and another begins takes a quarter longer (8192 x 8192 at rank 64: one sequence
// 51 us, seven 63 where the tiles are shared out by number), which up to kWideChunks chunks is weighed, by a chunk's first and last row.
constexpr int kWideChunks = 512;
struct WideShares {
  int weight[kWideChunks];
  int at[2];  // first tile, and the one behind the last
};
__device__ __forceinline__ void wide_share(WideShares& s, const ExpandWideParams& p) {
  const int cta = blockIdx.x, ctas = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long tiles = (long long)p.chunks * p.tiles;
  if (p.chunks > kWideChunks) {
    if (threadIdx.x < 2) s.at[threadIdx.x] = int(tiles * (cta + int(threadIdx.x)) / ctas);
    __syncthreads();
    return;
  }
  for (int c = threadIdx.x; c < p.chunks; c += blockDim.x)
    s.weight[c] = adapter_of(p.ids, c * 128, p.rows, p.L) == adapter_of(p.ids, min(c * 128 + 127, p.rows - 1), p.rows, p.L) ? 4 : 5;
  __syncthreads();
  if (warp == 0) {
    const int per = (p.chunks + 31) / 32, first = lane * per;
    int sum = 0;
    for (int c = first; c < min(first + per, p.chunks); ++c) sum += s.weight[c];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    const int total = __shfl_sync(0xffffffffu, before, 31);
    before -= sum;
    for (int i = 0; i < 2; ++i) {
      long long rest = (long long)total * p.tiles * (cta + i) / ctas - (long long)before * p.tiles;  // in weighted tiles, from the lane's first chunk on
      if (rest >= 0 && rest < (long long)sum * p.tiles) {
        int c = first;
        while (rest >= (long long)s.weight[c] * p.tiles) rest -= (long long)s.weight[c++] * p.tiles;
        s.at[i] = c * p.tiles + int(rest) / s.weight[c];
      }
    }
    if (lane == 0 && cta + 1 == ctas) s.at[1] = int(tiles);
  }
  __syncthreads();
}
template <bool TRANS>
__global__ void __launch_bounds__(ExpandWide<TRANS>::THREADS, 1)
adapter_expand_wide_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_out,
                           const ExpandWideParams p) {
  using Cfg = ExpandWide<TRANS>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ RowGroupsOf<Cfg::ROWS> groups;
  __shared__ WideShares shares;
  constexpr int BARS = 5 + 2 * Cfg::B_STAGES + 3 * Cfg::Y_STAGES;
  __shared__ __align__(8) uint64_t bars[BARS];
  __shared__ uint32_t tmem_slot, abort_word;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t a_full = smem_u32(bars);
  auto acc_full = [&](uint32_t i) { return smem_u32(bars + 1 + i); };
  auto acc_empty = [&](uint32_t i) { return smem_u32(bars + 3 + i); };
  auto b_full = [&](uint32_t i) { return smem_u32(bars + 5 + i); };
  auto b_empty = [&](uint32_t i) { return smem_u32(bars + 5 + Cfg::B_STAGES + i); };
  auto y_full = [&](uint32_t i) { return smem_u32(bars + 5 + 2 * Cfg::B_STAGES + i); };
  auto y_empty = [&](uint32_t i) { return smem_u32(bars + 5 + 2 * Cfg::B_STAGES + Cfg::Y_STAGES + i); };
  auto out_full = [&](uint32_t i) { return smem_u32(bars + 5 + 2 * Cfg::B_STAGES + 2 * Cfg::Y_STAGES + i); };
  WaitCtx ctx{&abort_word, p.status};
  if (threadIdx.x == 0) {
    for (int i = 0; i < BARS; ++i) mbar_init(smem_u32(bars + i), i == 0 || i == 3 || i == 4 || i >= BARS - Cfg::Y_STAGES ? Cfg::EPILOGUE_WARPS : 1);
    abort_word = 0u;
    fence_mbar_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_y);
    prefetch_tensormap(&map_out);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(&tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  wide_share(shares, p);
  const int u_end = shares.at[1];
  const int ksteps = p.Rp / 16;
  uint32_t a_phase = 0, bs = 0, b_phase = 0, ys = 0, y_phase = 0, acc = 0, acc_phase = 0;  // (each warp's own)
  for (int u = shares.at[0]; u < u_end;) {
    const int chunk = u / p.tiles, t0 = u - chunk * p.tiles, t1 = min(p.tiles, t0 + u_end - u);
    u += t1 - t0;
    const int row0 = chunk * Cfg::ROWS;
    __syncthreads();  // the groups of the chunk before have been read
    const int ngroups = group_rows(groups, p.ids, row0, p.rows, p.L);
    if (ngroups == 0 && p.in_place) continue;
    if (warp == 0) {
      for (int t = t0; t < t1; ++t) {
        const int c0 = t * Cfg::COLS;
        const int halves = c0 + 64 < p.C ? 2 : 1;
        if (p.has_y) {
          if (!mbar_wait(y_empty(ys), y_phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;  // given up: nothing more is issued
          if (elect_one()) {
            mbar_expect_tx(y_full(ys), uint32_t(halves * (Cfg::Y_BYTES / 2)));
            for (int h = 0; h < halves; ++h) tma_load_2d<1>(base + Cfg::Y_BASE + ys * Cfg::Y_BYTES + h * (Cfg::Y_BYTES / 2), &map_y, c0 + 64 * h, row0, y_full(ys));
          }
          __syncwarp();
          if (++ys == Cfg::Y_STAGES) { ys = 0; y_phase ^= 1u; }
        }
        for (int gi = 0; gi < ngroups; ++gi) {
          if (!mbar_wait(b_empty(bs), b_phase ^ 1u, ctx, WB_DEV_TIMEOUT_PRODUCER)) continue;
          if (elect_one()) {
            const uint32_t to = base + Cfg::B_BASE + bs * Cfg::B_BYTES;
            const int l = groups.adapter[gi];
            if constexpr (TRANS) {
              mbar_expect_tx(b_full(bs), uint32_t(halves * p.Rp * 128));
              for (int h = 0; h < halves; ++h) tma_load_2d<1>(to + h * (Cfg::B_BYTES / 2), &map_w, c0 + 64 * h, l * p.R, b_full(bs));
            } else {
              mbar_expect_tx(b_full(bs), Cfg::B_BYTES);
              tma_load_2d<1>(to, &map_w, 0, l * p.C + c0, b_full(bs));
            }
          }
          __syncwarp();
          if (++bs == Cfg::B_STAGES) { bs = 0; b_phase ^= 1u; }
        }
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = make_idesc_bf16_bt(Cfg::ROWS, Cfg::COLS) & ~(TRANS ? 0u : 1u << 16);  // B K-major, or MN-major
      if (ngroups > 0) {
        mbar_wait(a_full, a_phase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
        a_phase ^= 1u;
      }
      for (int t = t0; t < t1; ++t)
        for (int gi = 0; gi < ngroups; gi += 2) {
          mbar_wait(acc_empty(acc), acc_phase ^ 1u, ctx, WB_DEV_TIMEOUT_MMA_ACC);
          tc_fence_after_sync();
          const int ng = min(2, ngroups - gi);
          for (int i = 0; i < ng; ++i) {
            mbar_wait(b_full(bs), b_phase, ctx, WB_DEV_TIMEOUT_MMA_FULL);
            tc_fence_after_sync();
            if (elect_one()) {
              const uint32_t at = base + Cfg::B_BASE + bs * Cfg::B_BYTES;
              const uint64_t b = TRANS ? make_desc_mn_sw128(at, Cfg::B_BYTES / 2) : make_desc_k_sw128(at);
              for (int part = 0; part < kParts; ++part) {
                const uint64_t a = make_desc_k_sw128(base + part * (Cfg::A_BYTES / kParts));
                for (int k = 0; k < ksteps; ++k)
                  mma_f16<1>(tmem + (acc * 2 + i) * Cfg::COLS, a + uint64_t(k * 2), b + uint64_t(k * (TRANS ? 2048 >> 4 : 2)), idesc, (part > 0 || k > 0) ? 1u : 0u);
              }
              tc_commit<1>(b_empty(bs));
              if (i == ng - 1) tc_commit<1>(acc_full(acc));
            }
            __syncwarp();
            if (++bs == Cfg::B_STAGES) { bs = 0; b_phase ^= 1u; }
          }
          acc ^= 1u;
          if (acc == 0u) acc_phase ^= 1u;
        }
    } else if (warp < 2 + Cfg::EPILOGUE_WARPS) {
      const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane, id = groups.id[row];
      if (ngroups > 0) {  // the chunk's hidden vectors, pieces of 8 ranks (every MMA on those of the chunk before is complete: its sums were waited for)
        const int r = (int(threadIdx.x) - 64) >> 1;
        float v[4][8] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // all loads in flight together
          const int c = 2 * i + (threadIdx.x & 1);
          if (c * 8 < p.Rp && row0 + r < p.rows) read8<float>(p.hidden + (long long)(row0 + r) * p.Rp + c * 8, true, 8, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 2 * i + (threadIdx.x & 1);
          if (c * 8 >= p.Rp) break;
          uint32_t part[4][kParts];
#pragma unroll
          for (int j = 0; j < 4; ++j) split_pair(v[i][2 * j], v[i][2 * j + 1], part[j]);
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + q * (Cfg::A_BYTES / kParts) + r * 128 + ((c ^ (r & 7)) << 4)), "r"(part[0][q]), "r"(part[1][q]),
                         "r"(part[2][q]), "r"(part[3][q])
                         : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(a_full);
      }
      for (int t = t0; t < t1; ++t) {
        const int c0 = t * Cfg::COLS;
        mbar_wait(p.has_y ? y_full(ys) : y_empty(ys), p.has_y ? y_phase : y_phase ^ 1u, ctx, WB_DEV_TIMEOUT_EPILOGUE);
        const uint32_t mine = base + Cfg::Y_BASE + ys * Cfg::Y_BYTES + half * (Cfg::Y_BYTES / 2) + row * 128;
        auto at = [&](int piece_of_row) { return mine + uint32_t((piece_of_row ^ (row & 7)) << 4); };
        if (!p.has_y && id < 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at(i)), "r"(0u) : "memory");
        for (int gi = 0; gi < ngroups; gi += 2) {
          mbar_wait(acc_full(acc), acc_phase, ctx, WB_DEV_TIMEOUT_EPILOGUE);
          tc_fence_after_sync();
          const int ng = min(2, ngroups - gi);
          for (int i = 0; i < ng; ++i) {
            const bool hit = id == groups.adapter[gi + i];
            if (!__any_sync(0xffffffffu, hit)) continue;
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
              uint32_t v[32];
              tmem_ld_32x32(tmem + (uint32_t(quad * 32) << 16) + (acc * 2 + i) * Cfg::COLS + half * 64 + c, v);
              tmem_ld_wait();
              if (hit)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  uint32_t o[4] = {0u, 0u, 0u, 0u};
                  if (p.has_y) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(at(c / 8 + q)));
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    o[j] = pack_bf16x2(__uint_as_float(o[j] << 16) + __uint_as_float(v[8 * q + 2 * j]), __uint_as_float(o[j] & 0xffff0000u) + __uint_as_float(v[8 * q + 2 * j + 1]));
                  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at(c / 8 + q)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                }
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty(acc));
          acc ^= 1u;
          if (acc == 0u) acc_phase ^= 1u;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(out_full(ys));
        if (++ys == Cfg::Y_STAGES) { ys = 0; y_phase ^= 1u; }
      }
    } else {
      for (int t = t0; t < t1; ++t) {
        if (!mbar_wait(out_full(ys), y_phase, ctx, WB_DEV_TIMEOUT_EPILOGUE)) continue;  // given up
        if (lane == 0) {
          for (int h = 0; h < 2; ++h)
            if (t * Cfg::COLS + 64 * h < p.C) tma_store_2d(&map_out, base + Cfg::Y_BASE + ys * Cfg::Y_BYTES + h * (Cfg::Y_BYTES / 2), t * Cfg::COLS + 64 * h, row0);
          bulk_commit_group();
          bulk_wait_group_read<0>();
          mbar_arrive(y_empty(ys));
        }
        __syncwarp();
        if (++ys == Cfg::Y_STAGES) { ys = 0; y_phase ^= 1u; }
      }
    }
  }
  if (threadIdx.x == (2 + Cfg::EPILOGUE_WARPS) * 32) bulk_wait_group<0>();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
  }
}

// Rows of any alignment into rows of `pitch` (a multiple of 8) elements, zeros behind the last: what follows copies whole pieces.
__global__ void __launch_bounds__(256) adapter_align_kernel(const __nv_bfloat16* src, long long ld, int rows, int cols, __nv_bfloat16* dst, int pitch) {
  pdl_wait();
  pdl_launch_dependents();
  const int pieces = pitch / 8;
  const long long total = (long long)rows * pieces;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
    const int row = int(e / pieces), c = int(e - (long long)row * pieces) * 8;
    uint32_t r[4];
    load_bf16<8>(src + row * ld + c, false, cols - c, r);
    if (WB_CHECK(row < rows && c + 8 <= pitch, kCheckOutputIndex, (long long)row << 32 | c)) *reinterpret_cast<uint4*>(dst + e * 8) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

struct OuterSide {
  const __nv_bfloat16* z;       // [rows, C], pitch ldz
  const float* hidden;          // [rows][Rp]
  __nv_bfloat16* out;           // [L][C][R], or rank-major [L][R][C]
  long long ldz;
  int C, blocks, vec, rank_major;
};
struct OuterParams {
  OuterSide side[2];  // blocks of columns of the first, then of the second
  Ids ids;
  int rows, R, Rp, L;
};

// out_l[c, r] = sum over the rows t of adapter l of z[t, c] hidden[t, r]: B's gradient from g and A x, A's from x and B^T g.
// Grid (row splits = one cluster, blocks of 128 columns of both sides, adapters). A CTA picks the rows of its adapter out of its range of ids,
// in order, and adds up their outer products with MMAs whose k runs over the rows, from a ring of 64 rows a stage. The splits are
// added up through distributed shared memory, in their order. An MMA drops the bits of its f32 sum that do not fit, always towards zero, so that the
// products of 32 rows are summed by it and added to the others with rounding: over thousands of rows the sums would shrink by 3e-6 of themselves, several
// times what rounding costs. The warps stand side by side over the ranks first and over the columns where there are fewer ranks, so that a hidden number
// is split into its bf16 parts by as few of them as possible. Both sums of a backward pass are one launch: 4096 rows, 4096 + 4096 columns, rank 16
// 23 us (67 MB, 2.9 TB/s); bound by the start-up (ids, list, first loads), the barriers of the ring and the MMAs: a part takes 2 us of it. The CTAs of an
// adapter without rows look through all ids too: a call has (N + K) / 128 of them for every adapter of the pool.
constexpr int kOuterCols = 128;
constexpr int kOuterSegment = 4096;  // ids looked through at a time
template <int RT>
struct OuterTile {
  static constexpr int COLS = RT * 8;                                                     // ranks at a time
  static constexpr int WARPS_R = RT < 4 ? RT : 4, OCTETS = RT / WARPS_R;                  // warps over the ranks, eights of ranks of each
  static constexpr int WARPS_C = 4 / WARPS_R, MT = kOuterCols / 16 / WARPS_C;             // warps over the columns, sixteens of columns of each
  static constexpr int H_PIECES = COLS / 4;                                               // 16-byte pieces of a row of hidden numbers
  static constexpr int Z_BYTES = kChunkRows * kOuterCols * 2, H_BYTES = kChunkRows * COLS * 4, STAGE_BYTES = Z_BYTES + H_BYTES;
  static constexpr int STAGES = RT == 8 ? 3 : 4;
  static constexpr int SUM_PITCH = COLS + 4;  // 16-byte pieces of 8 neighbouring columns in different banks
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = RING_BYTES + kOuterSegment * 4;
  static_assert(2 * kOuterCols * SUM_PITCH * 4 <= RING_BYTES, "sums of the two halves of the rows");
  static_assert(kChunkRows * H_PIECES % kAdapterThreads == 0, "whole pieces of hidden numbers to a thread");
  // Place of 16-byte piece c of a row of hidden numbers: four lanes that read rows 2 apart meet different banks.
  __device__ static __forceinline__ uint32_t hidden_piece(int row, int c) { return uint32_t(row * H_PIECES + (c ^ ((((row >> 1) & 3) << 1) & (H_PIECES - 1)))) * 16; }
};

__device__ __forceinline__ void zero_fill(__nv_bfloat16* p, int n, int thread, int threads) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && n % 8 == 0)
    for (int i = thread; i < n / 8; i += threads) reinterpret_cast<uint4*>(p)[i] = make_uint4(0u, 0u, 0u, 0u);
  else
    for (int i = thread; i < n; i += threads) p[i] = __float2bfloat16_rn(0.f);
}

template <int RT>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_outer_kernel(const OuterParams p) {
  using Cfg = OuterTile<RT>;
  constexpr int STAGES = Cfg::STAGES, COLS = Cfg::COLS, OCTETS = Cfg::OCTETS, MT = Cfg::MT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int found[kAdapterWarps + 1];
  int* list = reinterpret_cast<int*>(smem + Cfg::RING_BYTES);
  const uint32_t base = smem_u32(smem);
  pdl_wait();
  pdl_launch_dependents();  // only now: this is the first kernel of a call that wants B's gradient alone
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int second = int(blockIdx.y) >= p.side[0].blocks;
  OuterSide side = p.side[0];  // (member by member: an index into the parameters would put them on the stack)
  if (second) side = p.side[1];
  const int c0 = (int(blockIdx.y) - (second ? p.side[0].blocks : 0)) * kOuterCols;
  const int l = blockIdx.z, splits = gridDim.x, split = blockIdx.x;
  const Ids& ids = p.ids;
  const int row_begin = int((long long)p.rows * split / splits), row_end = int((long long)p.rows * (split + 1) / splits);
  const int wr = (warp & 3) % Cfg::WARPS_R, wc = (warp & 3) / Cfg::WARPS_R, wk = warp >> 2;  // ranks, columns, 32 of a stage's 64 rows
  bool any = false;
  for (int n0 = 0; n0 < p.Rp; n0 += COLS) {
    float acc[MT][OCTETS][4] = {};
    for (int seg = row_begin; seg < row_end; seg += kOuterSegment) {
      // the segment's rows of this adapter, in order: a warp looks through a run of ids, then knows how many the warps before it found
      const int seg_end = min(row_end, seg + kOuterSegment);
      const int run = (seg_end - seg + kAdapterThreads - 1) / kAdapterThreads * 32;
      const int w0 = seg + warp * run, w1 = min(seg_end, w0 + run);
      constexpr int RUN = kOuterSegment / kAdapterThreads;  // 32-id steps of a full run
      unsigned hits[RUN];
      int mine = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RUN; ++i) {  // all of a lane's loads in flight together
        const int at = w0 + 32 * i + lane;
        hits[i] = at < w1 && adapter_of(ids, at, p.rows, p.L) == l;
      }
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        hits[i] = __ballot_sync(0xffffffffu, hits[i]);
        mine += __popc(hits[i]);
      }
      if (lane == 0) found[warp] = mine;
      __syncthreads();
      int at = 0, total = 0;
#pragma unroll
      for (int i = 0; i < kAdapterWarps; ++i) {
        at += i < warp ? found[i] : 0;
        total += found[i];
      }
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        if (hits[i] >> lane & 1u) list[at + __popc(hits[i] & ((1u << lane) - 1u))] = w0 + 32 * i + lane;
        at += __popc(hits[i]);
      }
      __syncthreads();
      const int steps = (total + kChunkRows - 1) / kChunkRows;
      any |= total > 0;
      // A thread brings the same pieces of every stage: column piece tid % 16 of rows tid / 16 + 16 i of z, and HN pieces of the hidden vectors
      constexpr int ZN = kChunkRows * (kOuterCols / 8) / kAdapterThreads, HN = kChunkRows * Cfg::H_PIECES / kAdapterThreads;
      const int zr = tid >> 4, zc = tid & 15;
      const int z_valid = min(8, side.C - c0 - zc * 8);
      const __nv_bfloat16* z_at = side.z + c0 + zc * 8;
      int next = 0;         // place in the list of the first row of the next load
      uint32_t to = base;   // its stage
      const bool fast = side.vec && c0 + kOuterCols <= side.C && n0 + COLS <= p.Rp;
      const int hr = tid / Cfg::H_PIECES, hc = tid % Cfg::H_PIECES;
      const float* h_at = side.hidden + n0 + hc * 4;
      constexpr int H_ROWS = kAdapterThreads / Cfg::H_PIECES;  // between the pieces of a thread
      auto load = [&]() {
        if (fast && next + kChunkRows <= total) {  // whole pieces of 64 rows
#pragma unroll
          for (int i = 0; i < ZN; ++i) cp_async16(to + piece<16>(zr + 16 * i, zc), z_at + list[next + zr + 16 * i] * side.ldz, true);
#pragma unroll
          for (int i = 0; i < HN; ++i)
            cp_async16(to + Cfg::Z_BYTES + Cfg::hidden_piece(hr + i * H_ROWS, hc), h_at + (long long)list[next + hr + i * H_ROWS] * p.Rp, true);
          cp_async_commit();
          next += kChunkRows;
          to = to == base + (STAGES - 1) * Cfg::STAGE_BYTES ? base : to + Cfg::STAGE_BYTES;
          return;
        }
#pragma unroll
        for (int i = 0; i < ZN; ++i) {
          const int in = next + zr + 16 * i;
          const bool real = in < total;
          copy8(to + piece<16>(zr + 16 * i, zc), real ? z_at + list[in] * side.ldz : z_at, side.z, side.vec != 0, real ? z_valid : 0);
        }
#pragma unroll
        for (int i = 0; i < HN; ++i) {
          const int r = hr + i * H_ROWS;
          const bool real = next + r < total && n0 + hc * 4 < p.Rp;
          cp_async16(to + Cfg::Z_BYTES + Cfg::hidden_piece(r, hc), real ? h_at + (long long)list[next + r] * p.Rp : side.hidden, real);
        }
        cp_async_commit();
        next += kChunkRows;
        to = to == base + (STAGES - 1) * Cfg::STAGE_BYTES ? base : to + Cfg::STAGE_BYTES;
      };
#pragma unroll
      for (int s = 0; s < STAGES - 1; ++s) {
        if (s < steps) load();
        else cp_async_commit();
      }
      uint32_t from = base;
      for (int step = 0; step < steps; ++step) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        if (step + STAGES - 1 < steps) load();
        else cp_async_commit();
        const int half = lane >> 4, in = lane & 15;
        // the lane's four rows of a rank (a column of the second operand) for either half of 16 rows: 2 t, 2 t + 1 and the same eight rows on
        uint32_t hf[2][OCTETS][2][kParts];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int o = 0; o < OCTETS; ++o) {
            const int rank = (wr * OCTETS + o) * 8 + g;
            const unsigned char* at = smem + (from - base) + Cfg::Z_BYTES + (32 * wk + 16 * k + 2 * t) * (COLS * 4) +
                                      (((rank >> 2) ^ ((2 * t) & (Cfg::H_PIECES - 1))) << 4) + (rank & 3) * 4;  // (hidden_piece of each of them)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              split_pair(*reinterpret_cast<const float*>(at + h * (COLS * 32)), *reinterpret_cast<const float*>(at + h * (COLS * 32) + COLS * 4), hf[k][o][h]);
          }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t za[2][4];  // matrices (k 0-7, c 0-7), (k 0-7, c 8-15), (k 8-15, c 0-7), (k 8-15, c 8-15)
#pragma unroll
          for (int k = 0; k < 2; ++k) ldsm4_trans(from + piece<16>(32 * wk + 16 * k + (in & 7) + half * 8, 2 * (wc * MT + m) + (in >> 3)), za[k]);
#pragma unroll
          for (int o = 0; o < OCTETS; ++o) {
            float sum[4] = {};
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int q = 0; q < kParts; ++q) mma_bf16(sum, za[k][0], za[k][1], za[k][2], za[k][3], hf[k][o][0][q], hf[k][o][1][q]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][o][e] += sum[e];
          }
        }
        from = from == base + (STAGES - 1) * Cfg::STAGE_BYTES ? base : from + Cfg::STAGE_BYTES;
      }
      cp_async_wait<0>();
    }
    if (splits == 1 && !any) {  // an adapter without rows
      const int cols = min(kOuterCols, side.C - c0);
      if (!WB_CHECK(l < p.L && cols > 0, kCheckOutputIndex, (long long)l << 32 | c0)) return;
      if (side.rank_major) {
        for (int r = warp; r < p.R; r += kAdapterWarps) zero_fill(side.out + ((long long)l * p.R + r) * side.C + c0, cols, lane, 32);
      } else {
        zero_fill(side.out + ((long long)l * side.C + c0) * p.R, cols * p.R, tid, kAdapterThreads);
      }
      return;
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);  // [2 halves of the rows][128 columns][SUM_PITCH]
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int o = 0; o < OCTETS; ++o)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sums[(wk * kOuterCols + 16 * (wc * MT + m) + g + (e >> 1) * 8) * Cfg::SUM_PITCH + (wr * OCTETS + o) * 8 + 2 * t + (e & 1)] = acc[m][o][e];
    __syncthreads();
    constexpr int QUADS = COLS / 4;  // four ranks of a column at a time
    float4* quads = reinterpret_cast<float4*>(sums);
    constexpr int QP = Cfg::SUM_PITCH / 4;
    for (int e = tid; e < kOuterCols * QUADS; e += kAdapterThreads) {  // the two halves of the rows
      float4& v = quads[e / QUADS * QP + e % QUADS];
      const float4 w = quads[(kOuterCols + e / QUADS) * QP + e % QUADS];
      v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
    }
    __syncthreads();
    if (splits > 1) {
      cluster_arrive();
      cluster_wait();
    }
    const int s0 = kOuterCols * split / splits, own = kOuterCols * (split + 1) / splits - s0;  // columns that this CTA finishes
    for (int e = tid; e < own * QUADS; e += kAdapterThreads) {
      const int c = s0 + (side.rank_major ? e % own : e / QUADS), q = side.rank_major ? e / own : e % QUADS;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (splits == 1) {
        v = quads[c * QP + q];
      } else {
        const uint32_t at = smem_u32(quads + c * QP + q);
        float4 part[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          part[s] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s < splits)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(part[s].x), "=f"(part[s].y), "=f"(part[s].z), "=f"(part[s].w)
                         : "r"(mapa_shared(at, s))
                         : "memory");
        }
#pragma unroll
        for (int s = 0; s < 8; ++s) v = make_float4(v.x + part[s].x, v.y + part[s].y, v.z + part[s].z, v.w + part[s].w);
      }
      const int r = n0 + 4 * q, col = c0 + c;
      if (col >= side.C || r >= p.R || !WB_CHECK(l < p.L && c >= 0 && c < kOuterCols, kCheckOutputIndex, (long long)l << 32 | col)) continue;
      const float f[4] = {v.x, v.y, v.z, v.w};
      if (side.rank_major) {
        __nv_bfloat16* to = side.out + ((long long)l * p.R + r) * side.C + col;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i < p.R) to[(long long)i * side.C] = __float2bfloat16_rn(f[i]);
      } else {
        __nv_bfloat16* to = side.out + ((long long)l * side.C + col) * p.R + r;
        if (p.R % 4 == 0 && (reinterpret_cast<uintptr_t>(side.out) & 7) == 0) {
          *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + i < p.R) to[i] = __float2bfloat16_rn(f[i]);
        }
      }
    }
    if (splits > 1) {  // nobody overwrites what others still read
      cluster_arrive();
      cluster_wait();
    }
    __syncthreads();
  }
}

}  // namespace wb
