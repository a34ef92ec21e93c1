// Low-rank adapters of many requests beside a shared projection, forward and backward:
//
//   out[t] = y[t] + s_l B_l (A_l x[t])        l = ids[t], A_l [R, K], B_l [N, R], bf16; rows without an adapter keep y
//   u[t]   = s_l B_l^T g[t]      dx[t] = A_l^T u[t]      dA_l = sum_t u[t] x[t]^T      dB_l = s_l sum_t g[t] (A_l x[t])^T
//
// Three kernels: `shrink` (rows times a wide matrix onto the ranks: A_l x, B_l^T g), `expand` (ranks onto wide rows: B_l h, A_l^T u) and
// `outer` (sums over the rows of an adapter). Each product is far below the tensor cores' rate at the ranks adapters have (2 R flops per
// two bytes of x), so they are bound by HBM for many rows and by latency for few, and what counts is that every row of x, y and g moves
// once, in whole 32-byte sectors.
//
// mma.sync m16n8k16 straight from global memory: an MMA adds over its 16 k in any order, so a lane may hold any 8 consecutive k of a row
// (one 16-byte load, two MMAs) as long as the other operand is permuted alike, and the columns of an output tile may be dealt to the lanes
// so that each has 8 neighbours. Operands whose contraction runs down the rows of memory (B_l^T, A_l^T, the outer products) are
// transposed by byte permutes of two registers.
//
// Rows are taken in chunks of 64 neighbours, and every CTA sorts the chunk's rows by adapter itself (64 compares a thread), so that no
// launch precedes it and ids need no order. A chunk of one sequence has one group of 64 rows; a decode step has groups of one row.
//
// The hidden vector h = A_l x (R numbers a row) is f32 in memory. It enters the second product as a sum of bf16 parts: two (relative
// error 2^-17) where the result is rounded to bf16, three (2^-25) where it stays f32.
#pragma once
#include <cuda_bf16.h>

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
struct RowGroups {
  int id[kChunkRows];
  int order[kChunkRows];      // rows of the chunk, those of one adapter together, in their order
  int start[kChunkRows + 1];  // first place of a group
  int adapter[kChunkRows];
  int leader[kChunkRows];
};

// Called by all threads of the CTA. Returns the number of groups. Ids outside [0, L) have no adapter.
template <typename IdT>
__device__ __forceinline__ int group_rows(RowGroups& g, const IdT* ids, int row0, int rows, int L) {
  const int t = threadIdx.x;
  int mine = -1;
  if (t < kChunkRows) {
    const long long id = row0 + t < rows ? (long long)ids[row0 + t] : -1;
    mine = id >= 0 && id < L ? int(id) : -1;
    g.id[t] = mine;
  }
  const int placed = __syncthreads_count(mine >= 0);
  int before = 0;
  bool first = mine >= 0;
  if (mine >= 0) {
#pragma unroll 8
    for (int j = 0; j < kChunkRows; ++j) {
      const int o = g.id[j];
      const bool same_before = o == mine && j < t;
      before += (o >= 0 && o < mine) || same_before;
      first &= !same_before;
    }
    g.order[before] = t;
  }
  if (t < kChunkRows) g.leader[t] = first ? mine : 0x7fffffff;
  const int groups = __syncthreads_count(first);
  if (first) {
    int at = 0;
#pragma unroll 8
    for (int j = 0; j < kChunkRows; ++j) at += g.leader[j] < mine;
    g.start[at] = before;
    g.adapter[at] = mine;
  }
  if (t == 0) g.start[groups] = placed;
  __syncthreads();
  return groups;
}

struct ShrinkParams {
  const __nv_bfloat16* x;  // [rows, K], pitch ldx
  const __nv_bfloat16* w;  // A_l [L][R][K], or (TRANS) B_l [L][K][R]
  const void* ids;
  float* hidden;  // [splits][rows][Rp]
  long long ldx;
  int rows, K, R, Rp, L, split_k;
  int x_vec, w_vec;  // 16-byte loads of x; vector loads of w
};

// hidden[split][t][r] = sum over the split's k of x[t, k] w_l[r, k]. Grid (splits, chunks, group lanes).
// The 8 warps of a CTA take blocks of KU * 32 k in turn and add up through shared memory, in warp order.
template <typename IdT, int RT, int MT, int KU, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_shrink_kernel(const ShrinkParams p) {
  __shared__ RowGroups groups;
  __shared__ float red[kAdapterWarps][16][RT * 8 + 2];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * kChunkRows;
  const int ngroups = group_rows(groups, static_cast<const IdT*>(p.ids), row0, p.rows, p.L);
  const int k0 = blockIdx.x * p.split_k, k1 = min(p.K, k0 + p.split_k);
  for (int gi = blockIdx.z; gi < ngroups; gi += gridDim.z) {
    const int end = groups.start[gi + 1];
    const __nv_bfloat16* w = p.w + (long long)groups.adapter[gi] * p.R * p.K;
    for (int first = groups.start[gi]; first < end; first += MT * 16) {
      const __nv_bfloat16* src[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = first + m * 16 + h * 8 + g;
          src[m][h] = at < end ? p.x + (long long)(row0 + groups.order[at]) * p.ldx : nullptr;
        }
      const int mtiles = min(MT, (end - first + 15) >> 4);
      for (int n0 = 0; n0 < p.Rp; n0 += RT * 8) {
        float acc[MT][RT][4] = {};
        for (int kb = k0 + warp * (KU * 32); kb < k1; kb += kAdapterWarps * KU * 32) {
          uint32_t xa[KU][MT][2][4];
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            const int k = kb + u * 32 + t * 8;
            const int valid = min(8, k1 - k);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (src[m][h] && valid > 0) load_bf16<8>(src[m][h] + k, p.x_vec != 0, valid, xa[u][m][h]);
                else xa[u][m][h][0] = xa[u][m][h][1] = xa[u][m][h][2] = xa[u][m][h][3] = 0u;
              }
          }
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            const int k = kb + u * 32 + t * 8;
            uint32_t wb_[RT][4];  // k pairs (0 1) (2 3) (4 5) (6 7) of the lane's eight
            if constexpr (!TRANS) {
              const int valid = min(8, k1 - k);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                const int r = n0 + i * 8 + g;
                if (r < p.R && valid > 0) load_bf16<8>(w + (long long)r * p.K + k, p.w_vec != 0, valid, wb_[i]);
                else wb_[i][0] = wb_[i][1] = wb_[i][2] = wb_[i][3] = 0u;
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
                  wb_[i][q] = i & 1 ? high_halves(raw[2 * q][i / 2], raw[2 * q + 1][i / 2]) : low_halves(raw[2 * q][i / 2], raw[2 * q + 1][i / 2]);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
              if (m < mtiles)
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                  for (int s = 0; s < 2; ++s)
                    mma_bf16(acc[m][i], xa[u][m][0][2 * s], xa[u][m][1][2 * s], xa[u][m][0][2 * s + 1], xa[u][m][1][2 * s + 1], wb_[i][2 * s],
                             wb_[i][2 * s + 1]);
          }
        }
        for (int m = 0; m < mtiles; ++m) {
          __syncthreads();
#pragma unroll
          for (int mm = 0; mm < MT; ++mm)
            if (mm == m)
#pragma unroll
              for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const int col = TRANS ? RT * (2 * t + (c & 1)) + i : i * 8 + 2 * t + (c & 1);
                  red[warp][g + (c >> 1) * 8][col] = acc[mm][i][c];
                }
          __syncthreads();
          for (int e = threadIdx.x; e < 16 * RT * 8; e += kAdapterThreads) {
            const int row = e / (RT * 8), col = e % (RT * 8), at = first + m * 16 + row;
            if (at >= end || n0 + col >= p.Rp) continue;
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < kAdapterWarps; ++v) sum += red[v][row][col];
            p.hidden[((long long)blockIdx.x * p.rows + row0 + groups.order[at]) * p.Rp + n0 + col] = sum;
          }
        }
        __syncthreads();
      }
    }
  }
}

struct ExpandParams {
  const __nv_bfloat16* w;  // B_l [L][C][R], or (TRANS) A_l [L][R][C]
  const void* ids;
  const float* scale;   // [L], or null
  const float* hidden;  // [splits][rows][Rp]
  const void* y;        // null: zeros
  void* out;
  long long ldy, ldo;
  int rows, C, R, Rp, L, splits, cols_per_cta;
  int io_vec, w_vec;
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

// `parts` bf16 values whose sum is v (each the rounding of what the ones before it leave).
template <int P>
__device__ __forceinline__ void split_bf16(float v, __nv_bfloat16 (&part)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    part[i] = __float2bfloat16_rn(v);
    const float rest = v - __bfloat162float(part[i]);
    v = fabsf(rest) < INFINITY ? rest : 0.f;  // an infinity or NaN is whole in its first part
  }
}

// out[t, c] = y[t, c] + s_l sum_r hidden[t, r] w_l[c, r]. Grid (column slices, chunks, group lanes). A warp takes 32 columns of all the
// rows of a group; a lane has 8 neighbouring columns of two rows. QN: steps of 16 ranks held in registers at a time.
template <typename IdT, typename T, int P, int QN, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_expand_kernel(const ExpandParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ RowGroups groups;
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(smem);  // [P][64][pitch]
  const int pitch = p.Rp + 8;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * kChunkRows;
  const int ngroups = group_rows(groups, static_cast<const IdT*>(p.ids), row0, p.rows, p.L);
  const int c_begin = blockIdx.x * p.cols_per_cta, c_end = min(p.C, c_begin + p.cols_per_cta);
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const int steps = p.Rp / 16;
  pdl_wait();
  for (int gi = blockIdx.z; gi < ngroups; gi += gridDim.z) {
    const int first = groups.start[gi], count = groups.start[gi + 1] - first;
    const int l = groups.adapter[gi];
    const float s = p.scale ? p.scale[l] : 1.f;
    __syncthreads();
    const int mtiles = (count + 15) >> 4;
    for (int e = threadIdx.x; e < mtiles * 16 * p.Rp; e += kAdapterThreads) {
      const int row = e / p.Rp, r = e - row * p.Rp;
      float v = 0.f;
      if (row < count) {
        const float* h = p.hidden + (long long)(row0 + groups.order[first + row]) * p.Rp + r;
        for (int i = 0; i < p.splits; ++i) v += h[(long long)i * p.rows * p.Rp];
      }
      __nv_bfloat16 part[P];
      split_bf16<P>(v * s, part);
#pragma unroll
      for (int i = 0; i < P; ++i) hs[(i * kChunkRows + row) * pitch + r] = part[i];
    }
    __syncthreads();
    const __nv_bfloat16* w = p.w + (long long)l * p.R * p.C;
    for (int c0 = c_begin + warp * kExpandCols; c0 < c_end; c0 += kAdapterWarps * kExpandCols) {
      uint32_t wf[4][QN][2];
      auto load_w = [&](int q0) {
#pragma unroll
        for (int q = 0; q < QN; ++q) {
          const int r = (q0 + q) * 16 + 4 * t;
          if constexpr (!TRANS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = c0 + 8 * (g >> 1) + 2 * i + (g & 1);
              if (c < p.C && r < p.R) load_bf16<4>(w + (long long)c * p.R + r, p.w_vec != 0 && r + 4 <= p.R, p.R - r, wf[i][q]);
              else wf[i][q][0] = wf[i][q][1] = 0u;
            }
          } else {
            uint32_t raw[4][2];
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
      };
      if (steps <= QN) load_w(0);
      const int col = c0 + 8 * t;
      const int valid = p.C - col;
      const bool whole = p.io_vec && valid >= 8;
      for (int m = 0; m < mtiles; ++m) {
        int row[2];
        float old[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = m * 16 + h * 8 + g;
          row[h] = at < count ? row0 + groups.order[first + at] : -1;
#pragma unroll
          for (int i = 0; i < 8; ++i) old[h][i] = 0.f;
          if (y && row[h] >= 0 && valid > 0) read8<T>(y + row[h] * p.ldy + col, whole, valid, old[h]);
        }
        float acc[4][4] = {};
        for (int q0 = 0; q0 < steps; q0 += QN) {
          if (steps > QN) load_w(q0);
#pragma unroll
          for (int q = 0; q < QN; ++q) {
            if (q0 + q >= steps) break;
            const __nv_bfloat16* at = hs + (m * 16 + g) * pitch + (q0 + q) * 16 + 4 * t;
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const uint2 lo = *reinterpret_cast<const uint2*>(at + i * kChunkRows * pitch);
              const uint2 hi = *reinterpret_cast<const uint2*>(at + (i * kChunkRows + 8) * pitch);
#pragma unroll
              for (int n = 0; n < 4; ++n) mma_bf16(acc[n], lo.x, hi.x, lo.y, hi.y, wf[n][q][0], wf[n][q][1]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (row[h] < 0 || valid <= 0) continue;
          float v[8];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int at = TRANS ? 4 * j + n : 2 * n + j;
              v[at] = old[h][at] + acc[n][2 * h + j];
            }
          write8<T>(out + row[h] * p.ldo + col, whole, valid, v);
        }
      }
    }
  }
  if (blockIdx.z == 0 && p.out != p.y) {  // rows without an adapter
    for (int row = warp; row < min(kChunkRows, p.rows - row0); row += kAdapterWarps) {
      if (groups.id[row] >= 0) continue;
      for (int c = c_begin + lane * 8; c < c_end; c += 256) {
        const int valid = p.C - c;
        float v[8] = {};
        if (y) read8<T>(y + (row0 + row) * p.ldy + c, p.io_vec && valid >= 8, valid, v);
        write8<T>(out + (row0 + row) * p.ldo + c, p.io_vec && valid >= 8, valid, v);
      }
    }
  }
}

struct OuterParams {
  const __nv_bfloat16* z;  // [rows, C], pitch ldz
  const float* hidden;     // [splits][rows][Rp]
  const float* scale;      // [L], or null
  const int* list;         // rows sorted by adapter
  const int* owner;        // adapter of every entry of the list
  const int* listed;       // entries of the list
  float* part;             // [row splits][L][C][Rp], or (RANK_MAJOR) [row splits][L][Rp][C]
  long long ldz;
  int rows, C, R, Rp, L, splits;
  int z_vec;
};

__device__ __forceinline__ int first_of(const int* owner, int n, int l) {  // first entry whose adapter is at least l
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (owner[mid] < l) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// part[split][l][c][r] = sum over the split's rows t of adapter l of z[t, c] s_l hidden[t, r]. Grid (column blocks of 256, L, row splits).
// A warp takes 32 columns; RT tiles of 8 ranks at a time. The hidden vectors of 64 rows are in shared memory, two rows to a word, as
// two bf16 parts.
template <int RT, bool RANK_MAJOR>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_outer_kernel(const OuterParams p) {
  constexpr int P = 2, PITCH = RT * 8 + 4;
  __shared__ uint32_t hs[P][kChunkRows / 2][PITCH];
  __shared__ int rows_of[kChunkRows];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int l = blockIdx.y;
  const int n = *p.listed;
  const int seg0 = first_of(p.owner, n, l), seg1 = first_of(p.owner, n, l + 1);
  const int blocks = (seg1 - seg0 + kChunkRows - 1) / kChunkRows;
  const int b0 = int((long long)blocks * blockIdx.z / gridDim.z), b1 = int((long long)blocks * (blockIdx.z + 1) / gridDim.z);
  const float s = p.scale ? p.scale[l] : 1.f;
  const int c = blockIdx.x * (kAdapterWarps * 32) + warp * 32 + 4 * g;  // the lane's four columns
  const bool whole = p.z_vec && c + 4 <= p.C;
  for (int n0 = 0; n0 < p.Rp; n0 += RT * 8) {
    float acc[2][RT][4] = {};
    for (int b = b0; b < b1; ++b) {
      const int first = seg0 + b * kChunkRows, count = min(kChunkRows, seg1 - first);
      __syncthreads();
      if (threadIdx.x < kChunkRows) rows_of[threadIdx.x] = threadIdx.x < count ? p.list[first + threadIdx.x] : -1;
      __syncthreads();
      for (int e = threadIdx.x; e < kChunkRows / 2 * RT * 8; e += kAdapterThreads) {
        const int pair = e / (RT * 8), r = e - pair * (RT * 8);
        uint32_t word[P] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = rows_of[2 * pair + h];
          if (row < 0 || n0 + r >= p.Rp) continue;
          float v = 0.f;
          for (int i = 0; i < p.splits; ++i) v += p.hidden[((long long)i * p.rows + row) * p.Rp + n0 + r];
          __nv_bfloat16 part[P];
          split_bf16<P>(v * s, part);
#pragma unroll
          for (int i = 0; i < P; ++i) word[i] |= uint32_t(__bfloat16_as_ushort(part[i])) << (16 * h);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) hs[i][pair][r] = word[i];
      }
      __syncthreads();
      if (c - 4 * g < p.C) {  // the warp's first column
#pragma unroll
        for (int k = 0; k < kChunkRows / 16; ++k) {
          if (k * 16 >= count) break;
          uint32_t raw[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = rows_of[k * 16 + 4 * t + i];
            if (row >= 0 && c < p.C) load_bf16<4>(p.z + row * p.ldz + c, whole, p.C - c, raw[i]);
            else raw[i][0] = raw[i][1] = 0u;
          }
          uint32_t za[2][4];  // column tiles: columns 4 g and 4 g + 1, 4 g + 2 and 4 g + 3
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            za[m][0] = low_halves(raw[0][m], raw[1][m]);
            za[m][1] = high_halves(raw[0][m], raw[1][m]);
            za[m][2] = low_halves(raw[2][m], raw[3][m]);
            za[m][3] = high_halves(raw[2][m], raw[3][m]);
          }
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int q = 0; q < P; ++q) {
              const uint32_t h0 = hs[q][8 * k + 2 * t][i * 8 + g], h1 = hs[q][8 * k + 2 * t + 1][i * 8 + g];
#pragma unroll
              for (int m = 0; m < 2; ++m) mma_bf16(acc[m][i], za[m][0], za[m][1], za[m][2], za[m][3], h0, h1);
            }
        }
      }
    }
    float* part = p.part + ((long long)blockIdx.z * p.L + l) * p.C * p.Rp;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = c + 2 * m + (e >> 1), r = n0 + i * 8 + 2 * t + (e & 1);
          if (col < p.C && r < p.Rp) part[RANK_MAJOR ? (long long)r * p.C + col : (long long)col * p.Rp + r] = acc[m][i][e];
        }
    __syncthreads();
  }
}

// out[l][i][j] = sum over the splits, in their order, of part[split][l][i][j]; j runs over `inner` of `pitch` entries of a row.
__global__ void __launch_bounds__(256)
adapter_reduce_kernel(const float* part, int splits, int L, int outer_used, int outer_n, int inner, int pitch, __nv_bfloat16* out) {
  pdl_launch_dependents();
  pdl_wait();
  const long long per = (long long)outer_used * inner, total = per * L;
  const long long stride = (long long)L * outer_n * pitch;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
    const int l = int(e / per);
    const long long in = e - l * per;
    const int i = int(in / inner), j = int(in - (long long)i * inner);
    const float* src = part + ((long long)l * outer_n + i) * pitch + j;
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += src[s * stride];
    out[e] = __float2bfloat16_rn(v);
  }
}

}  // namespace wb
