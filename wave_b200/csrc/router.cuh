// Router of an expert MLP with what its training needs, forward and backward, and the gradient of the weighted sum behind it.
//
//   p[t] = softmax(logits[t])      ids[t] = the k largest logits, the lower expert first among equals, NaN above all
//   weight[t, j] = p[t, ids[t, j]]  (renormalised: over their sum)
//   counts[e] = pairs (t, j) with ids[t, j] = e      loss = E sum_e counts[e] / (k n) * sum_t p[t, e] / n      n = rows that are not masked
//   d loss / d p[t, e] = E counts[e] / (k n^2)       d logits = p (dp - sum p dp)
//
// A warp takes a row, a lane the experts e = lane + 32 i. Everything is in f32 in registers: the row is read once. The sums over the rows
// (p per expert, counts) are kept per lane over all the rows of a warp, added up by CTA, then over the CTAs by a second launch, each in a
// fixed order; up to kRouterOneCta rows there is one CTA and one launch. Bound by latency: 8192 rows of 256 f32 logits are 8 MB.
#pragma once
#include <cuda_bf16.h>

#include "ptx.cuh"

namespace wb {

constexpr int kRouterMaxExperts = 256;
constexpr int kRouterMaxTopK = 32;
constexpr int kRouterWarps = 8;
constexpr int kRouterOneCta = 64;
constexpr int kRouterMaxCtas = 296;

struct RouterParams {
  const void* logits;
  const uint8_t* mask;   // [rows], null: no row is masked
  const void* given;     // choices made elsewhere (ids, as given_i64 says), or null: chosen here
  long long ld;
  int rows, E, top_k, renormalize, given_i64;
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

// exp(z - max) of a row's logits, and 1 / their sum.
template <typename T, int EV>
__device__ __forceinline__ float softmax_row(const T* row, int E, int lane, float (&z)[EV], float (&x)[EV]) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EV; ++i) {
    const int e = lane + 32 * i;
    z[i] = e < E ? logit_value(row + e) : -INFINITY;
    mx = (mx != mx || z[i] != z[i]) ? __int_as_float(0x7fc00000) : fmaxf(mx, z[i]);
  }
  mx = warp_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < EV; ++i) {
    x[i] = lane + 32 * i < E ? expf(z[i] - mx) : 0.f;
    sum += x[i];
  }
  return 1.f / warp_sum(sum);
}

// What the partial sums become, by a CTA: thread (e, q) of THREADS / EP slices adds up every so-manieth CTA's sums of expert e, then the
// slices are added in order.
template <int THREADS>
__device__ __forceinline__ void router_finish(const RouterParams& p, int ctas, double (*sums)[THREADS], int (*counts)[THREADS]) {
  const int EP = (p.E + 31) / 32 * 32, slices = THREADS / EP;
  const int e = threadIdx.x % EP, q = threadIdx.x / EP;
  double sum = 0.0;
  int count = 0;
  if (q < slices && e < p.E) {
#pragma unroll 8
    for (int c = q; c < ctas; c += slices) {
      sum += p.part_p[c * p.E + e];
      count += p.part_n[c * (p.E + 1) + e];
    }
  }
  int n = 0;
  for (int c = threadIdx.x; c < ctas; c += THREADS) n += p.part_n[c * (p.E + 1) + p.E];
  (*sums)[threadIdx.x] = sum;
  (*counts)[threadIdx.x] = count;
  __syncthreads();
  double mine = 0.0;
  if (threadIdx.x < p.E) {
    for (int i = 1; i < slices; ++i) {
      sum += (*sums)[i * EP + threadIdx.x];
      count += (*counts)[i * EP + threadIdx.x];
    }
    p.counts[threadIdx.x] = count;
    mine = sum * count;
  }
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mine += __shfl_xor_sync(0xffffffffu, mine, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    (*sums)[threadIdx.x >> 5] = mine;
    (*counts)[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    n = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      total += (*sums)[w];
      n += (*counts)[w];
    }
    const double unit = n > 0 ? p.E / (double(p.top_k) * n * n) : 0.0;
    *p.unit = float(unit);
    *p.loss = float(total * unit);
  }
}

template <typename T, int EV>
__global__ void __launch_bounds__(kRouterWarps * 32)
router_kernel(const RouterParams p) {
  __shared__ float sum_p[kRouterWarps][EV * 32];
  __shared__ int sum_n[EV * 32 + 1];
  __shared__ double sums[kRouterWarps * 32];
  __shared__ int counts[kRouterWarps * 32];
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
    if (!kept) {
      if (!p.given && lane < p.top_k) { ids[lane] = -1; weight[lane] = 0.f; }
      continue;
    }
    ++seen;
    float z[EV], x[EV];
    const float inv = softmax_row<T, EV>(static_cast<const T*>(p.logits) + (long long)t * p.ld, p.E, lane, z, x);
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
    uint32_t key[EV];
#pragma unroll
    for (int i = 0; i < EV; ++i) key[i] = lane + 32 * i < p.E ? choice_key(z[i]) : 0u;
    int chosen = -1;     // lane j: the j-th choice, and its p
    float chosen_p = 0.f;
    for (int j = 0; j < p.top_k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < EV; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      uint32_t e = 0xffffffffu;
#pragma unroll
      for (int i = EV - 1; i >= 0; --i)
        if (key[i] == best && best != 0u) e = lane + 32 * i;
      e = __reduce_min_sync(0xffffffffu, e);
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < EV; ++i)
        if (e == uint32_t(lane + 32 * i)) {
          key[i] = 0u;
          v = x[i];
        }
      v = __shfl_sync(0xffffffffu, v, e & 31);
      if (lane == j) { chosen = int(e); chosen_p = v; }
    }
    float scale = inv;
    if (p.renormalize) scale = 1.f / warp_sum(chosen_p);
    if (lane < p.top_k) {
      ids[lane] = chosen;
      weight[lane] = chosen_p * scale;
      atomicAdd(&sum_n[chosen], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < EV; ++i) sum_p[warp][lane + 32 * i] = acc[i];
  if (lane == 0) atomicAdd(&sum_n[EV * 32], seen);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kRouterWarps * 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRouterWarps; ++w) sum += sum_p[w][e];
    p.part_p[blockIdx.x * p.E + e] = sum;
    p.part_n[blockIdx.x * (p.E + 1) + e] = sum_n[e];
  }
  if (threadIdx.x == 0) p.part_n[blockIdx.x * (p.E + 1) + p.E] = sum_n[EV * 32];
  if (gridDim.x == 1) {
    __syncthreads();
    router_finish<kRouterWarps * 32>(p, 1, &sums, &counts);
  }
}

__global__ void __launch_bounds__(1024) router_finish_kernel(const RouterParams p, int ctas) {
  __shared__ double sums[1024];
  __shared__ int counts[1024];
  pdl_launch_dependents();
  pdl_wait();
  router_finish<1024>(p, ctas, &sums, &counts);
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
};

template <typename T, int EV>
__global__ void __launch_bounds__(kRouterWarps * 32)
router_grad_kernel(const RouterGradParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float unit = p.g_loss ? *p.g_loss * *p.unit : 0.f;
  float loss_dp[EV];
#pragma unroll
  for (int i = 0; i < EV; ++i) loss_dp[i] = lane + 32 * i < p.E ? unit * p.counts[lane + 32 * i] : 0.f;
  for (int t = blockIdx.x * kRouterWarps + warp; t < p.rows; t += gridDim.x * kRouterWarps) {
    T* out = static_cast<T*>(p.g_logits) + (long long)t * p.ldg;
    if (p.mask && !p.mask[t]) {
      for (int e = lane; e < p.E; e += 32) out[e] = T(0.f);
      continue;
    }
    float z[EV], x[EV], dp[EV];
    const float inv = softmax_row<T, EV>(static_cast<const T*>(p.logits) + (long long)t * p.ld, p.E, lane, z, x);
#pragma unroll
    for (int i = 0; i < EV; ++i) { x[i] *= inv; dp[i] = loss_dp[i]; }
    if (p.ids && p.g_weight) {
      const int mine = lane < p.top_k ? p.ids[(long long)t * p.top_k + lane] : -1;
      float gw = lane < p.top_k ? p.g_weight[(long long)t * p.top_k + lane] : 0.f;
      if (p.renormalize) {
        float q = 0.f;  // p of the lane's choice
        for (int j = 0; j < p.top_k; ++j) {
          const int e = __shfl_sync(0xffffffffu, mine, j);
          float v = 0.f;
#pragma unroll
          for (int i = 0; i < EV; ++i)
            if (e == lane + 32 * i) v = x[i];
          v = __shfl_sync(0xffffffffu, v, e & 31);
          if (lane == j) q = v;
        }
        const float total = warp_sum(q);
        const float dot = warp_sum(q * gw) / total;
        gw = (gw - dot) / total;
      }
      for (int j = 0; j < p.top_k; ++j) {
        const int e = __shfl_sync(0xffffffffu, mine, j);
        const float v = __shfl_sync(0xffffffffu, gw, j);
#pragma unroll
        for (int i = 0; i < EV; ++i)
          if (e == lane + 32 * i) dp[i] += v;
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < EV; ++i) dot += x[i] * dp[i];
    dot = warp_sum(dot);
#pragma unroll
    for (int i = 0; i < EV; ++i)
      if (lane + 32 * i < p.E) out[lane + 32 * i] = T(x[i] * (dp[i] - dot));
  }
}

// g_weight[t, j] = sum_c g[t, c] y[row_of[t, j], c]: the gradient of moe_combine by its weights; 0 for dropped pairs. A CTA takes a token:
// its row of g is read once, next to the rows of four slots at a time. Bound by HBM: (k + 1) rows read per token.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128)
combine_grad_kernel(const T* g, long long ldg, const T* y, long long ldy, const int* row_of, int top_k, int cols, float* g_weight) {
  __shared__ float part[4][4];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = blockIdx.x;
  for (int j0 = 0; j0 < top_k; j0 += 4) {
    int row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) row[j] = j0 + j < top_k ? row_of[t * top_k + j0 + j] : -1;
    float acc[4] = {};
    for (int c = threadIdx.x * 8; c < cols; c += 1024) {
      float a[8], b[4][8];
      const int valid = cols - c;
      read8<T>(g + t * ldg + c, VEC, valid, a);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row[j] >= 0) read8<T>(y + row[j] * ldy + c, VEC, valid, b[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row[j] >= 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[j] += a[i] * b[j][i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[j] = warp_sum(acc[j]);
      if (lane == 0) part[warp][j] = acc[j];
    }
    __syncthreads();
    if (threadIdx.x < 4 && j0 + threadIdx.x < top_k)
      g_weight[t * top_k + j0 + threadIdx.x] = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
    __syncthreads();
  }
}

}  // namespace wb
