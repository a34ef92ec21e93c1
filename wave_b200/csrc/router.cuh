// Router of an expert MLP with what its training needs, forward and backward, and the gradient of the weighted sum behind it.
//
//   p[t] = softmax(logits[t])      ids[t] = the k largest logits, the lower expert first among equals, NaN above all
//   weight[t, j] = p[t, ids[t, j]]  (renormalised: over their sum)
//   counts[e] = pairs (t, j) with ids[t, j] = e      loss = E sum_e counts[e] / (k n) * sum_t p[t, e] / n      n = rows that are not masked
//   d loss / d p[t, e] = E counts[e] / (k n^2)       d logits = p (dp - sum p dp)
//
// A warp takes a row, a lane EV neighbouring experts. Everything is in f32 in registers: the row is read once. The largest of what is left is one
// warp-wide integer maximum a choice; the lowest lane that holds it is the lowest expert. The sums over the rows (p per expert, counts) are kept per
// lane over all the rows of a warp, added up by CTA, then over the CTAs by a second launch (one cluster, 32 experts a CTA), each in a fixed
// order; up to kRouterOneCta rows there is one CTA and one launch. Bound by latency and by issue slots (62 % in the forward kernel, which makes k
// dependent warp-wide maxima a row): 8192 rows of 256 f32 logits (8 MB), top 8, 32 us for the three launches of a training step; 16 rows of 8 3.7 us.
#pragma once
#include <cuda_bf16.h>

#include "ptx.cuh"

namespace wb {

constexpr int kRouterMaxExperts = 256;
constexpr int kRouterMaxTopK = 32;
constexpr int kRouterWarps = 8;
constexpr int kRouterOneCta = 64;
constexpr int kRouterMaxCtas = 592;  // four per SM

struct RouterParams {
  const void* logits;
  const uint8_t* mask;   // [rows], null: no row is masked
  const void* given;     // choices made elsewhere (ids, as given_i64 says), or null: chosen here
  long long ld;
  int rows, E, top_k, renormalize, given_i64;
  int vec;               // rows start on 16 bytes, E is a multiple of a lane's experts
  float* weight;         // [rows, top_k] (chosen here)
  int* ids;              // [rows, top_k] (chosen here)
  float* part_p;         // [CTAs][E]
  int* part_n;           // [CTAs][E + 1]: counts, rows
  int* counts;           // [E]
  float* unit;           // E / (k n^2): what a count adds to the gradient of p; 0 where no row counts
  float* loss;
};

__device__ __forceinline__ float logit_value(const float* p) { return *p; }
__device__ __forceinline__ float logit_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Order of the choice: integers in the order of the values, every NaN above the infinity; 0 for what may not be chosen.
__device__ __forceinline__ uint32_t choice_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == 0.f) v = 0.f;  // -0 and 0 are equal
  const uint32_t b = __float_as_uint(v);
  return ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = (v != v || w != w) ? __int_as_float(0x7fc00000) : fmaxf(v, w);
  }
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row's logits, EV neighbouring experts to a lane (-inf behind the last expert), exp(z - max), and 1 / the sum of those.
template <typename T, int EV>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, bool vec, float (&z)[EV]) {
  const int e0 = lane * EV;
  if (vec && EV * sizeof(T) >= 8) {  // E is a multiple of EV, and rows start on 16 bytes
#pragma unroll
    for (int i = 0; i < EV; ++i) z[i] = -INFINITY;
    if (e0 < E) {
      if constexpr (EV * sizeof(T) >= 8) {
        constexpr int WORDS = EV * sizeof(T) / 4;
        uint32_t w[WORDS];
        if constexpr (WORDS >= 4) {
#pragma unroll
          for (int i = 0; i < WORDS / 4; ++i) {
            const uint4 v = *(reinterpret_cast<const uint4*>(row + e0) + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(row + e0);
          w[0] = v.x; w[1] = v.y;
        }
#pragma unroll
        for (int i = 0; i < EV; ++i) {
          if constexpr (sizeof(T) == 4) z[i] = __uint_as_float(w[i]);
          else z[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EV; ++i) z[i] = e0 + i < E ? logit_value(row + e0 + i) : -INFINITY;
  }
}
template <int EV>
__device__ __forceinline__ float softmax_row(const float (&z)[EV], int E, int lane, float (&x)[EV], float& mx) {
  mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EV; ++i) mx = (mx != mx || z[i] != z[i]) ? __int_as_float(0x7fc00000) : fmaxf(mx, z[i]);
  mx = warp_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < EV; ++i) {
    x[i] = lane * EV + i < E ? expf(z[i] - mx) : 0.f;
    sum += x[i];
  }
  return 1.f / warp_sum(sum);
}

// What the partial sums become. 32 experts (and this CTA's place among `blocks` of them), 32 threads each: a thread adds up every 32nd CTA's sums
// in their order, the 32 are added in order, and the loss over the CTAs of the cluster in order. 1024 threads.
__global__ void __launch_bounds__(1024) router_finish_kernel(const RouterParams p, int ctas) {
  __shared__ double sums[32][33];
  __shared__ int counts[32][33];
  __shared__ double total;
  __shared__ int rows[32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;  // a warp reads 32 neighbouring experts of a CTA's sums
  double sum = 0.0;
  int count = 0, n = 0;
  constexpr int MOST = (kRouterMaxCtas + 31) / 32;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int c = warp + 32 * i;
    if (c < ctas && e < p.E) {
      sum += p.part_p[c * p.E + e];
      count += p.part_n[c * (p.E + 1) + e];
    }
    if (c < ctas && lane == 0) n += p.part_n[c * (p.E + 1) + p.E];
  }
  sums[warp][lane] = sum;
  counts[warp][lane] = count;
  if (lane == 0) rows[warp] = n;
  __syncthreads();
  if (warp == 0) {
    sum = 0.0;
    count = n = 0;
    for (int i = 0; i < 32; ++i) {
      sum += sums[i][lane];
      count += counts[i][lane];
      n += rows[i];
    }
    if (e < p.E && WB_CHECK(count >= 0, kCheckOutputIndex, e)) p.counts[e] = count;
    double mine = e < p.E ? sum * count : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) {
      total = mine;
      rows[0] = n;
    }
  }
  const int blocks = gridDim.x;
  __syncthreads();
  if (blocks > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double all = 0.0;
    for (int i = 0; i < blocks; ++i) {
      double v = total;
      if (i > 0) asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(smem_u32(&total), i)) : "memory");
      all += v;
    }
    n = rows[0];
    const double unit = n > 0 ? p.E / (double(p.top_k) * n * n) : 0.0;
    *p.unit = float(unit);
    *p.loss = float(all * unit);
  }
  if (blocks > 1) {  // nobody leaves while its total may still be read
    cluster_arrive();
    cluster_wait();
  }
}

template <typename T, int EV>
__global__ void __launch_bounds__(kRouterWarps * 32)
router_kernel(const RouterParams p) {
  __shared__ float sum_p[kRouterWarps][EV * 32];
  __shared__ int sum_n[EV * 32 + 1];
  __shared__ double share[kRouterWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < EV * 32 + 1; e += kRouterWarps * 32) sum_n[e] = 0;
  __syncthreads();
  float acc[EV] = {};
  int seen = 0;
  for (int t = blockIdx.x * kRouterWarps + warp; t < p.rows; t += gridDim.x * kRouterWarps) {
    const bool kept = !p.mask || p.mask[t];
    int* ids = p.ids + (long long)t * p.top_k;
    float* weight = p.weight + (long long)t * p.top_k;
    float z[EV], x[EV], mx;
    load_row<T, EV>(static_cast<const T*>(p.logits) + (long long)t * p.ld, p.E, lane, p.vec != 0, z);
    if (!kept) {
      if (!p.given && lane < p.top_k) { ids[lane] = -1; weight[lane] = 0.f; }
      continue;
    }
    ++seen;
    const float inv = softmax_row<EV>(z, p.E, lane, x, mx);
#pragma unroll
    for (int i = 0; i < EV; ++i) acc[i] += x[i] * inv;
    if (p.given) {
      for (int j = lane; j < p.top_k; j += 32) {
        const long long at = (long long)t * p.top_k + j;
        const long long e = p.given_i64 ? static_cast<const long long*>(p.given)[at] : static_cast<const int*>(p.given)[at];
        if (e >= 0 && e < p.E) atomicAdd(&sum_n[e], 1);
      }
      continue;
    }
    uint32_t key[EV], best = 0;
#pragma unroll
    for (int i = 0; i < EV; ++i) {
      key[i] = lane * EV + i < p.E ? choice_key(z[i]) : 0u;
      best = max(best, key[i]);
    }
    int chosen = -1;     // lane j: the j-th choice, and its exponential
    float chosen_x = 0.f;
    for (int j = 0; j < p.top_k; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const int owner = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
      int at = 0;
      float v = 0.f;
      if (lane == owner) {
#pragma unroll
        for (int i = EV - 1; i >= 0; --i)
          if (key[i] == top) { at = i; v = x[i]; }
        best = 0;
#pragma unroll
        for (int i = 0; i < EV; ++i) {
          if (i == at) key[i] = 0u;
          best = max(best, key[i]);
        }
      }
      at = __shfl_sync(0xffffffffu, at, owner);
      v = __shfl_sync(0xffffffffu, v, owner);
      if (lane == j) { chosen = owner * EV + at; chosen_x = v; }
    }
    float scale = inv;
    if (p.renormalize) scale = 1.f / warp_sum(chosen_x);
    if (lane < p.top_k && WB_CHECK(t < p.rows && chosen >= 0 && chosen < p.E, kCheckOutputIndex, (long long)t << 32 | unsigned(chosen))) {
      ids[lane] = chosen;
      weight[lane] = chosen_x * scale;
      atomicAdd(&sum_n[chosen], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < EV; ++i) sum_p[warp][lane * EV + i] = acc[i];
  if (lane == 0) atomicAdd(&sum_n[EV * 32], seen);
  __syncthreads();
  double mine = 0.0;
  for (int e = threadIdx.x; e < p.E; e += kRouterWarps * 32) {  // (E is at most the number of threads)
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRouterWarps; ++w) sum += sum_p[w][e];
    if (gridDim.x == 1) {
      p.counts[e] = sum_n[e];
      mine = double(sum) * sum_n[e];
    } else {
      if (!WB_CHECK(blockIdx.x < kRouterMaxCtas, kCheckPartialSlot, blockIdx.x)) break;
      p.part_p[blockIdx.x * p.E + e] = sum;
      p.part_n[blockIdx.x * (p.E + 1) + e] = sum_n[e];
    }
  }
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) p.part_n[blockIdx.x * (p.E + 1) + p.E] = sum_n[EV * 32];
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) share[warp] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int w = 0; w < kRouterWarps; ++w) total += share[w];
    const int n = sum_n[EV * 32];
    const double unit = n > 0 ? p.E / (double(p.top_k) * n * n) : 0.0;
    *p.unit = float(unit);
    *p.loss = float(total * unit);
  }
}

struct RouterGradParams {
  const void* logits;
  const uint8_t* mask;
  const int* ids;          // [rows, top_k] as chosen by the router, or null: no gradient of the weights
  const float* g_weight;   // [rows, top_k], or null
  const float* g_loss;     // device scalar, or null
  const int* counts;
  const float* unit;
  void* g_logits;          // [rows, E], pitch ldg
  long long ld, ldg;
  int rows, E, top_k, renormalize;
  int vec;                 // as RouterParams, of g_logits too
};

template <typename T, int EV>
__global__ void __launch_bounds__(kRouterWarps * 32)
router_grad_kernel(const RouterGradParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = lane * EV;
  const float unit = p.g_loss ? *p.g_loss * *p.unit : 0.f;
  float loss_dp[EV];
#pragma unroll
  for (int i = 0; i < EV; ++i) loss_dp[i] = e0 + i < p.E ? unit * p.counts[e0 + i] : 0.f;
  for (int t = blockIdx.x * kRouterWarps + warp; t < p.rows; t += gridDim.x * kRouterWarps) {
    T* out = static_cast<T*>(p.g_logits) + (long long)t * p.ldg;
    const T* row = static_cast<const T*>(p.logits) + (long long)t * p.ld;
    const bool kept = !p.mask || p.mask[t];
    float d[EV] = {};
    if (kept) {
      const bool weights = p.ids && p.g_weight;
      float z[EV], x[EV], mx, gw = 0.f, zj = 0.f;
      int mine = -1;  // the lane's choice
      load_row<T, EV>(row, p.E, lane, p.vec != 0, z);
      if (weights && lane < p.top_k) {
        mine = p.ids[(long long)t * p.top_k + lane];
        gw = p.g_weight[(long long)t * p.top_k + lane];
        if (mine >= 0) zj = logit_value(row + mine);
      }
      const float inv = softmax_row<EV>(z, p.E, lane, x, mx);
#pragma unroll
      for (int i = 0; i < EV; ++i) { x[i] *= inv; d[i] = loss_dp[i]; }
      if (weights) {
        if (p.renormalize) {
          const float q = mine >= 0 ? expf(zj - mx) * inv : 0.f;  // p of the lane's choice
          const float total = warp_sum(q);
          const float dot = warp_sum(q * gw) / total;
          gw = (gw - dot) / total;
        }
        for (int j = 0; j < p.top_k; ++j) {
          const int at = __shfl_sync(0xffffffffu, mine, j) - e0;
          const float v = __shfl_sync(0xffffffffu, gw, j);
#pragma unroll
          for (int i = 0; i < EV; ++i)
            if (at == i) d[i] += v;
        }
      }
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < EV; ++i) dot += x[i] * d[i];
      dot = warp_sum(dot);
#pragma unroll
      for (int i = 0; i < EV; ++i) d[i] = x[i] * (d[i] - dot);
    }
    if constexpr (EV == 8) {
      if (p.vec) {
        if (e0 < p.E && WB_CHECK(t < p.rows && e0 + 8 <= p.E, kCheckOutputIndex, (long long)t << 32 | e0)) write8<T>(out + e0, true, 8, d);
        continue;
      }
    }
#pragma unroll
    for (int i = 0; i < EV; ++i)
      if (e0 + i < p.E && WB_CHECK(t < p.rows, kCheckOutputIndex, (long long)t << 32 | (e0 + i))) out[e0 + i] = T(d[i]);
  }
}

// out[t] = sum_j weight[t, j] y[row_of[t, j]] in slot order, for bf16 rows that start on 16 bytes: a CTA takes a token, all its pairs (SLOTS at a time)
// and two pieces of their rows are in flight behind the row numbers. The same sums as moe_combine_kernel, which has a thread per piece of 8
// columns, in the same order. 4096 x 4096 in pairs 15 us (101 MB), where a thread per piece took 23; narrow rows stay with the other, whose CTAs
// share tokens, and so do few tokens of wide rows, which it has in flight all at once (wb200_moe_combine has the rule).
template <int SLOTS>
__global__ void __launch_bounds__(128)
combine_token_kernel(const __nv_bfloat16* y, long long ldy, const int* row_of, const float* weight, int top_k, int cols, __nv_bfloat16* out, long long ldo) {
  constexpr int U = 2;
  pdl_wait();
  pdl_launch_dependents();
  const long long t = blockIdx.x;
  int row[SLOTS];
  float w[SLOTS];
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    row[j] = j < top_k ? row_of[t * top_k + j] : -1;
    w[j] = j < top_k ? weight[t * top_k + j] : 0.f;
  }
  for (int c = threadIdx.x * 8; c < cols; c += U * 1024) {
    uint4 b[SLOTS][U];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u)
        b[j][u] = row[j] >= 0 && c + u * 1024 < cols ? *reinterpret_cast<const uint4*>(y + row[j] * ldy + c + u * 1024) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * 1024 >= cols) break;
      float acc[8] = {};
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        if (row[j] < 0) continue;
        float v[8];
        read8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(&b[j][u]), true, 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += w[j] * v[i];
      }
      if (WB_CHECK(c + u * 1024 + 8 <= cols, kCheckOutputIndex, t << 32 | (c + u * 1024))) write8<__nv_bfloat16>(out + t * ldo + c + u * 1024, true, 8, acc);
    }
  }
}

// g_weight[t, j] = sum_c g[t, c] y[row_of[t, j], c]: the gradient of moe_combine by its weights; 0 for dropped pairs. A CTA takes a token:
// its row of g is read once, next to the rows of SLOTS pairs at a time, two pieces of every row in flight. Bound by HBM: (k + 1) rows read per
// token, 4096 x 4096 in pairs 18 us (101 MB, 5.6 TB/s; with one piece in flight 34).
template <typename T, bool VEC, int SLOTS>
__global__ void __launch_bounds__(128)
combine_grad_kernel(const T* g, long long ldg, const T* y, long long ldy, const int* row_of, int top_k, int cols, float* g_weight) {
  constexpr int U = 2;
  __shared__ float part[4][SLOTS];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = blockIdx.x;
  for (int j0 = 0; j0 < top_k; j0 += SLOTS) {
    int row[SLOTS];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) row[j] = j0 + j < top_k ? row_of[t * top_k + j0 + j] : -1;
    float acc[SLOTS] = {};
    if constexpr (VEC && sizeof(T) == 2) {
      for (int c = threadIdx.x * 8; c < cols; c += U * 1024) {
        uint4 a[U], b[SLOTS][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool there = c + u * 1024 < cols;
          a[u] = there ? *reinterpret_cast<const uint4*>(g + t * ldg + c + u * 1024) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int j = 0; j < SLOTS; ++j)
            b[j][u] = there && row[j] >= 0 ? *reinterpret_cast<const uint4*>(y + row[j] * ldy + c + u * 1024) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float av[8];
          read8<T>(reinterpret_cast<const T*>(&a[u]), true, 8, av);
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) {
            if (row[j] < 0 || c + u * 1024 >= cols) continue;
            float bv[8];
            read8<T>(reinterpret_cast<const T*>(&b[j][u]), true, 8, bv);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[j] += av[i] * bv[i];
          }
        }
      }
    } else {
      for (int c = threadIdx.x * 8; c < cols; c += 1024) {
        float a[8], b[SLOTS][8];
        const int valid = cols - c;
        read8<T>(g + t * ldg + c, VEC, valid, a);
#pragma unroll
        for (int j = 0; j < SLOTS; ++j)
          if (row[j] >= 0) read8<T>(y + row[j] * ldy + c, VEC, valid, b[j]);
#pragma unroll
        for (int j = 0; j < SLOTS; ++j)
          if (row[j] >= 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[j] += a[i] * b[j][i];
      }
    }
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      acc[j] = warp_sum(acc[j]);
      if (lane == 0) part[warp][j] = acc[j];
    }
    __syncthreads();
    if (threadIdx.x < SLOTS && j0 + threadIdx.x < top_k && WB_CHECK(t < gridDim.x, kCheckOutputIndex, t))
      g_weight[t * top_k + j0 + threadIdx.x] = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
    __syncthreads();
  }
}

}  // namespace wb
