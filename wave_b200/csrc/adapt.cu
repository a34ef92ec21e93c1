// C entry points of what is trained and served beside frozen MXFP4 weights: low-rank adapters, the input gradient of a linear layer,
// the router of an expert MLP with its balance loss, and the gradient of the weighted combine.
#include "../../include/wave_b200.h"
#include "host.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <initializer_list>
#include <iterator>
#include <mutex>

#include "adapters.cuh"
#include "input_grad_sm100.cuh"
#include "router.cuh"

namespace {

using wbhost::fail;

constexpr int kTargetCtas = 296;  // two per SM of a B200

bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool words_aligned(std::initializer_list<const void*> pointers) {  // to four bytes (a null pointer is)
  return std::all_of(pointers.begin(), pointers.end(), [](const void* p) { return aligned_to(p, 4); });
}
int div_up(long long a, long long b) { return int((a + b - 1) / b); }
int rank_pad(int R) { return (R + 15) / 16 * 16; }
int chunks_of(int rows) { return div_up(rows, wb::kChunkRows); }
// The kernels for few rows (taken 32 at a time) are those for groups of a few rows: a group's rows share the loads of its adapter but not its arithmetic.
// us, few / many, K = N = 4096: rank 16, 1 row 5.2 / 6.4, 8 rows of one adapter 7.6 / 6.4, 32 rows of one 20.3 / 7.1, of eight 8.0 / 8.8, of 64
// 8.9 / 12.8; rank 64, 4 rows of one adapter 8.8 / 8.6, 64 rows of 16 13.6 / 16.4.
bool few_rows(int rows, int L) { return rows <= 64 && rows < 8ll * L; }

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// Lets a kernel have up to BYTES of dynamic shared memory, once per device.
template <auto Kernel, int BYTES = 200 * 1024>
int allow_smem() {
  static bool done[wbhost::kMaxDevices] = {};
  int dev = 0;
  WB_HOST_CUDA(cudaGetDevice(&dev));
  if (!done[dev]) {
    WB_HOST_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES));
    done[dev] = true;
  }
  return WB200_OK;
}

// ------------------------------------------------------------------------------------------
// adapters
// ------------------------------------------------------------------------------------------
// A launch whose grid.x is one cluster.
template <typename... P, typename... A>
cudaError_t launch_clusters(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = grid.x;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = grid.x > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// The smallest power of two, at most `most` and 8 (a cluster), with which `units` come to two CTAs per SM.
int splits_for(long long units, int most) {
  int s = 1;
  while (s < 8 && 2 * s <= most && units * s < kTargetCtas * 2 / 3) s *= 2;
  return s;
}
// CTAs that share the groups of a chunk. Four at least where there are adapters enough: a chunk in which one sequence ends and another begins has two
// groups, and as one CTA's work it took twice as long as the others (8192 rows of 6 sequences, K = N = 8192, rank 64: 255 us for both products with
// one lane, 192 with four); a CTA without a group leaves at once.
int group_lanes(int rows, int L, long long others) {
  return few_rows(rows, L) ? std::min({rows, L, wb::kFewRows}) : int(std::max<long long>(std::min(4, L), std::min<long long>(std::min(wb::kChunkRows, L), kTargetCtas / others)));
}

struct AdapterCall {
  wb::Ids ids;
  int rows, R, Rp, L;
  cudaStream_t stream;
  int* status;
  int sms;
};

template <int RT, bool TRANS>
int launch_shrink(const wb::ShrinkParams& p, bool few, dim3 grid, cudaStream_t s) {
  if (few) {
    WB_HOST_CUDA(launch_clusters(wb::adapter_shrink_few_kernel<RT, TRANS>, grid, wb::kAdapterThreads, 0, s, p));
    return WB200_OK;
  }
  constexpr auto kernel = wb::adapter_shrink_tile_kernel<RT, TRANS>;
  if (int rc = allow_smem<kernel>()) return rc;
  WB_HOST_CUDA(launch_clusters(kernel, grid, wb::kAdapterThreads, wb::ShrinkTile<RT>::SMEM_BYTES, s, p));
  return WB200_OK;
}
template <bool TRANS>
int launch_shrink_ranks(const wb::ShrinkParams& p, bool few, dim3 grid, cudaStream_t s) {
  return p.Rp <= 16 ? launch_shrink<2, TRANS>(p, few, grid, s) : p.Rp <= 32 ? launch_shrink<4, TRANS>(p, few, grid, s) : launch_shrink<8, TRANS>(p, few, grid, s);
}

template <int N, bool TRANS>
int launch_shrink_wide(const AdapterCall& c, wb::ShrinkParams p, int chunks) {
  using Cfg = wb::ShrinkWide<N, TRANS>;
  const int splits = splits_for(chunks, std::max(1, p.K / 256));
  p.split_k = div_up(div_up(p.K, splits), 64) * 64;
  CUtensorMap x, w;
  if (int rc = wbhost::tensor_map(&x, p.x, p.K, p.rows, (unsigned long long)p.ldx * 2, 64, Cfg::ROWS, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return rc;
  const unsigned long long inner = TRANS ? p.R : p.K, outer = (unsigned long long)p.L * (TRANS ? p.K : p.R);
  if (int rc = wbhost::tensor_map(&w, p.w, inner, outer, inner * 2, 64, TRANS ? 64 : N, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  constexpr auto kernel = wb::adapter_shrink_wide_kernel<N, TRANS>;
  if (int rc = allow_smem<kernel>()) return rc;
  const int lanes = int(std::max<long long>(1, std::min<long long>(div_up(std::min(Cfg::ROWS, c.L), 2), kTargetCtas / ((long long)chunks * splits))));
  WB_HOST_CUDA(launch_clusters(kernel, dim3(splits, chunks, lanes), wb::kAdapterThreads, Cfg::SMEM_BYTES, c.stream, x, w, p, c.status));
  return WB200_OK;
}
// The tensor cores take 2048 rows or more, and any number of more than 32 ranks. us of both products, ring of copies / tensor cores, K = N = 4096, three sequences:
// rank 16, 1024 rows 15.8 / 18.4, 2048 rows 26.0 / 22.8, 8192 rows 45.0 / 46.3; rank 64, 256 rows 18.0 / 17.0, 2048 rows 37.6 / 28.2; 4096 rows of 64 mixed
// adapters at rank 16 430 / 423. Rows of few ranks are short pieces for the copy engine (trans): 4096 rows of rank 16 with gradients 74 / 79 with both.
bool wide_shrink(const AdapterCall& c, const wb::ShrinkParams& p, bool trans) {
  return p.x_vec && aligned_to(p.w, 16) && p.K % 64 == 0 && (!trans || p.R % 8 == 0) && (long long)p.L * std::max(p.K, p.R) < 0x7fffffff &&
         (c.Rp > 32 || (c.rows >= 2048 && !trans));
}

// hidden [rows][Rp] = rows of x onto the ranks, scaled. trans: w is [L][K][R].
int run_shrink(const AdapterCall& c, const __nv_bfloat16* x, long long ldx, int K, const __nv_bfloat16* w, bool trans, const float* scale, float* hidden) {
  wb::ShrinkParams p;
  p.x = x; p.w = w; p.ids = c.ids; p.scale = scale; p.hidden = hidden; p.ldx = ldx;
  p.rows = c.rows; p.K = K; p.R = c.R; p.Rp = c.Rp; p.L = c.L;
  const bool few = few_rows(c.rows, c.L);
  p.x_vec = aligned_to(x, 16) && ldx % 8 == 0 && ldx >= (K + 7) / 8 * 8;  // (a piece that K ends in is there, zeros behind)
  if (!few && wide_shrink(c, p, trans)) {
    const int wide = div_up(c.rows, 128);
    return trans        ? launch_shrink_wide<64, true>(c, p, wide)
           : c.Rp <= 16 ? launch_shrink_wide<16, false>(c, p, wide)
           : c.Rp <= 32 ? launch_shrink_wide<32, false>(c, p, wide)
                        : launch_shrink_wide<64, false>(c, p, wide);
  }
  const int chunks = few ? div_up(c.rows, wb::kFewRows) : chunks_of(c.rows);
  const int splits = few ? splits_for(1, std::max(1, K / 512)) : splits_for(chunks, std::max(1, K / 256));
  p.split_k = div_up(div_up(K, splits), 64) * 64;
  const int vec = !trans ? 8 : !few ? 8 : c.Rp <= 16 ? 2 : c.Rp <= 32 ? 4 : 8;  // elements of a load of w
  p.w_vec = aligned_to(w, 2 * vec) && (trans ? c.R : K) % vec == 0;
  const dim3 grid(splits, chunks, group_lanes(c.rows, c.L, (long long)chunks * splits));
  return trans ? launch_shrink_ranks<true>(p, few, grid, c.stream) : launch_shrink_ranks<false>(p, few, grid, c.stream);
}

template <typename T, int QN, bool TRANS, bool FAST, bool EXACT>
int launch_expand_tile(const wb::ExpandParams& p, dim3 grid, cudaStream_t s) {
  constexpr auto kernel = wb::adapter_expand_tile_kernel<T, QN, TRANS, FAST, EXACT>;
  const size_t smem = size_t(wb::kChunkRows) * wb::expand_pitch(p.Rp, FAST && EXACT && QN % 2 == 0) * 2 + (FAST ? wb::expand_ring_bytes(sizeof(T), EXACT) : 0);
  if (int rc = smem > 24 * 1024 ? allow_smem<kernel>() : WB200_OK) return rc;
  WB_HOST_CUDA(launch(kernel, grid, wb::kAdapterThreads, smem, s, p));
  return WB200_OK;
}
// Lanes that share a column of B in the kernel for few rows of whole ranks, 0 where that is not taken.
int whole_pieces(const wb::ExpandParams& p) {
  return p.w_vec && p.R == p.Rp && (p.R == 16 || p.R == 32 || p.R == 64) ? p.R / 8 : p.w_vec && p.R == 8 ? 1 : 0;
}

template <typename T, bool TRANS>
int launch_expand(const wb::ExpandParams& p, bool few, dim3 grid, cudaStream_t s) {
  if (few) {
    if constexpr (!TRANS)
      if (const int pieces = whole_pieces(p)) {
        auto kernel = pieces == 1   ? wb::adapter_expand_few_whole_kernel<T, 1>
                      : pieces == 2 ? wb::adapter_expand_few_whole_kernel<T, 2>
                      : pieces == 4 ? wb::adapter_expand_few_whole_kernel<T, 4>
                                    : wb::adapter_expand_few_whole_kernel<T, 8>;
        WB_HOST_CUDA(launch(kernel, grid, wb::kAdapterThreads, 0, s, p));
        return WB200_OK;
      }
    WB_HOST_CUDA(launch(wb::adapter_expand_few_kernel<T, TRANS>, grid, wb::kAdapterThreads, size_t(8) * p.Rp * 4, s, p));
    return WB200_OK;
  }
  const int steps = p.Rp / 16;
  if (p.io_vec && p.w_vec && p.C % 8 == 0 && (TRANS || steps % 2 == 1 || p.R % 8 == 0))
    return steps == 1   ? launch_expand_tile<T, 1, TRANS, true, true>(p, grid, s)
           : steps == 2 ? launch_expand_tile<T, 2, TRANS, true, true>(p, grid, s)
           : steps == 4 ? launch_expand_tile<T, 4, TRANS, true, true>(p, grid, s)
                        : launch_expand_tile<T, 4, TRANS, true, false>(p, grid, s);
  return steps == 1 ? launch_expand_tile<T, 1, TRANS, false, true>(p, grid, s) : launch_expand_tile<T, 2, TRANS, false, false>(p, grid, s);
}

template <bool TRANS>
int launch_expand_wide(const AdapterCall& c, const wb::ExpandParams& e) {
  using Cfg = wb::ExpandWide<TRANS>;
  wb::ExpandWideParams p;
  p.ids = e.ids; p.hidden = e.hidden; p.rows = e.rows; p.C = e.C; p.R = e.R; p.Rp = e.Rp; p.L = e.L;
  p.chunks = div_up(e.rows, Cfg::ROWS); p.tiles = div_up(e.C, Cfg::COLS);
  p.has_y = e.y != nullptr; p.in_place = e.out == e.y; p.status = c.status;
  constexpr auto bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  constexpr auto swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
  constexpr auto promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  CUtensorMap w, y, out;
  const unsigned long long inner = TRANS ? e.C : e.R, outer = (unsigned long long)e.L * (TRANS ? e.R : e.C);
  if (int rc = wbhost::tensor_map(&w, e.w, inner, outer, inner * 2, 64, TRANS ? e.Rp : Cfg::COLS, bf16, swizzle)) return rc;
  if (int rc = wbhost::tensor_map(&out, e.out, e.C, e.rows, (unsigned long long)e.ldo * 2, 64, Cfg::ROWS, bf16, swizzle)) return rc;
  y = out;
  if (e.y)
    if (int rc = wbhost::tensor_map(&y, e.y, e.C, e.rows, (unsigned long long)e.ldy * 2, 64, Cfg::ROWS, bf16, swizzle, promotion)) return rc;
  constexpr auto kernel = wb::adapter_expand_wide_kernel<TRANS>;
  if (int rc = allow_smem<kernel, Cfg::SMEM_BYTES>()) return rc;
  const dim3 grid(unsigned(std::min<long long>(c.sms, (long long)p.chunks * p.tiles)));
  WB_HOST_CUDA(launch(kernel, grid, Cfg::THREADS, Cfg::SMEM_BYTES, c.stream, w, y, out, p));
  return WB200_OK;
}
// The tensor cores take more than 32 ranks where y and out are larger than L2. us of both products with the shrinking one on the tensor cores, rank 64:
// 4096 x 4096 41.1 / 44.6, 8192 x 4096 70.3 / 60.9, 16384 x 8192 230 / 165; rank 32, 16384 x 8192 169 / 156, 8192 x 8192 91.6 / 89.3, 8192 x 4096 53.6 / 56.7.
bool wide_expand(const AdapterCall& c, const wb::ExpandParams& p, bool trans, bool f32) {
  return !f32 && p.io_vec && aligned_to(p.w, 16) && p.C % 8 == 0 && p.Rp <= 64 && p.R % (trans ? 16 : 8) == 0 && (long long)p.L * std::max(p.C, p.R) < 0x7fffff00 && p.Rp > 32 && (long long)c.rows * p.C >= 1 << 25;
}

// out = y + ranks onto C columns.
int run_expand(const AdapterCall& c, const __nv_bfloat16* w, bool trans, const float* hidden, const void* y, long long ldy, void* out, long long ldo, bool f32, int C) {
  wb::ExpandParams p;
  p.w = w; p.ids = c.ids; p.hidden = hidden; p.y = y; p.out = out; p.ldy = ldy; p.ldo = ldo;
  p.rows = c.rows; p.C = C; p.R = c.R; p.Rp = c.Rp; p.L = c.L;
  const bool few = few_rows(c.rows, c.L);
  const int chunks = few ? div_up(c.rows, wb::kFewRows) : chunks_of(c.rows);
  // one wave of CTAs where that leaves each several rounds of its 256 columns: what a CTA does before its first column (grouping, hidden vectors)
  // takes as long as a few rounds
  p.cols_per_cta = few ? 2 * wb::kAdapterThreads : div_up(div_up(C, std::max(1, kTargetCtas / chunks)), 256) * 256;
  const size_t esz = f32 ? 4 : 2;
  p.io_vec = aligned_to(out, 16) && ldo * esz % 16 == 0 && (!y || (aligned_to(y, 16) && ldy * esz % 16 == 0));
  p.io_pairs = !f32 && C % 2 == 0 && aligned_to(out, 4) && ldo % 2 == 0 && (!y || (aligned_to(y, 4) && ldy % 2 == 0));
  if (!few && wide_expand(c, p, trans, f32)) return trans ? launch_expand_wide<true>(c, p) : launch_expand_wide<false>(c, p);
  const int vec = few ? (trans ? 2 : 8) : !trans && c.R % 8 == 0 ? 8 : 4;  // elements of a load of w
  p.w_vec = aligned_to(w, 2 * vec) && (trans ? C : c.R) % (trans && few ? 4 : vec) == 0;
  if (few && !trans)
    if (const int pieces = whole_pieces(p)) p.cols_per_cta = wb::few_whole_steps(pieces) * wb::kAdapterThreads / pieces;
  const int slices = div_up(C, p.cols_per_cta);
  const dim3 grid(slices, chunks, group_lanes(c.rows, c.L, (long long)chunks * slices));
  using bf16 = __nv_bfloat16;
  return trans ? launch_expand<bf16, true>(p, few, grid, c.stream)
         : f32 ? launch_expand<float, false>(p, few, grid, c.stream) : launch_expand<bf16, false>(p, few, grid, c.stream);
}

template <int RT>
int launch_outer(const wb::OuterParams& p, dim3 grid, cudaStream_t s) {
  constexpr auto kernel = wb::adapter_outer_kernel<RT>;
  if (int rc = allow_smem<kernel>()) return rc;
  WB_HOST_CUDA(launch_clusters(kernel, grid, wb::kAdapterThreads, wb::OuterTile<RT>::SMEM_BYTES, s, p));
  return WB200_OK;
}

// Either side may be left out (out null); the splits, and with them the order of the sums, do not depend on that.
int run_outer(const AdapterCall& c, wb::OuterSide first, wb::OuterSide second) {
  wb::OuterParams p;
  p.side[0] = first;
  p.side[1] = second;
  for (wb::OuterSide& side : p.side) {
    side.blocks = side.out ? div_up(side.C, wb::kOuterCols) : 0;
    side.vec = aligned_to(side.z, 16) && side.ldz % 8 == 0 && side.ldz >= (side.C + 7) / 8 * 8;
  }
  p.ids = c.ids;
  p.rows = c.rows; p.R = c.R; p.Rp = c.Rp; p.L = c.L;
  const int blocks = p.side[0].blocks + p.side[1].blocks;
  const long long both = (long long)div_up(first.C, wb::kOuterCols) + div_up(second.C, wb::kOuterCols);
  const dim3 grid(splits_for(both * c.L, chunks_of(c.rows)), blocks, c.L);
  return c.Rp <= 16 ? launch_outer<2>(p, grid, c.stream) : c.Rp <= 32 ? launch_outer<4>(p, grid, c.stream) : launch_outer<8>(p, grid, c.stream);
}

int check_adapters(const char* what, int rows, int K, int N, int R, int L) {
  if (rows <= 0 || K <= 0 || N <= 0 || R <= 0 || L <= 0)
    return fail(WB200_ERR_INVALID_ARG, "%s: rows = %d, K = %d, N = %d, rank = %d, adapters = %d", what, rows, K, N, R, L);
  if (K % 8) return fail(WB200_ERR_INVALID_ARG, "%s: K = %d is not a multiple of 8", what, K);
  if (R > 256) return fail(WB200_ERR_UNSUPPORTED, "%s: rank %d is above 256", what, R);
  if (rows > 4000000) return fail(WB200_ERR_UNSUPPORTED, "%s: %d rows in one call", what, rows);
  if ((long long)div_up(N, 128) + div_up(K, 128) > 65535) return fail(WB200_ERR_UNSUPPORTED, "%s: K = %d and N = %d are too wide", what, K, N);
  return WB200_OK;
}

// ------------------------------------------------------------------------------------------
// input gradient
// ------------------------------------------------------------------------------------------
// CTAs to a tile (1: 128 x 128, a pair: 256 x 256) and slices of the sum over N (a cluster of cg * slices CTAs to a tile).
struct InputGradLayout {
  int cg, slices;
};
constexpr InputGradLayout kInputGradLayouts[] = {{2, 1}, {1, 1}, {2, 2}, {1, 2}, {2, 3}, {1, 3}, {2, 4}, {1, 4}, {1, 6}, {1, 8}};

template <int CG>
int input_grad_config(int slices, cudaStream_t stream, cudaLaunchConfig_t* cfg, cudaLaunchAttribute (&attr)[2]) {
  using Cfg = wb::InputGradCfg<CG>;
  static bool done[wbhost::kMaxDevices] = {};
  int dev = 0;
  WB_HOST_CUDA(cudaGetDevice(&dev));
  if (!done[dev]) {
    WB_HOST_CUDA(cudaFuncSetAttribute(wb::input_grad_kernel<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    done[dev] = true;
  }
  *cfg = {};
  cfg->gridDim = dim3(CG * slices, 1, 1);
  cfg->blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg->dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG * slices;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 2;
  return WB200_OK;
}

// How many clusters of every layout run at one time on the current device.
int input_grad_resident(const int** out) {
  static int resident[wbhost::kMaxDevices][std::size(kInputGradLayouts)] = {};
  static std::mutex mu;
  int dev = 0;
  WB_HOST_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  if (!resident[dev][0])
    for (int i = int(std::size(kInputGradLayouts)) - 1; i >= 0; --i) {
      cudaLaunchConfig_t cfg;
      cudaLaunchAttribute attr[2];
      const InputGradLayout l = kInputGradLayouts[i];
      if (int rc = l.cg == 2 ? input_grad_config<2>(l.slices, nullptr, &cfg, attr) : input_grad_config<1>(l.slices, nullptr, &cfg, attr)) return rc;
      int n = 0;
      cfg.numAttrs = 1;
      WB_HOST_CUDA(l.cg == 2 ? cudaOccupancyMaxActiveClusters(&n, wb::input_grad_kernel<2>, &cfg) : cudaOccupancyMaxActiveClusters(&n, wb::input_grad_kernel<1>, &cfg));
      resident[dev][i] = n > 0 ? n : -1;
    }
  *out = resident[dev];
  return WB200_OK;
}

// The layout of least estimated time. Measured (us): a step of 64 N takes 0.42 with either tile, a launch 4 on top of its steps, and each round
// of sliced tiles 10.5, for filling the ring, reading the accumulators and adding them up. 16 x 14336 x 4096: one CTA a tile 88, four slices
// 30; 600 x 4000 x 2048: pairs 31, two slices 25; 2048^3: pairs 21, two slices 38.
int input_grad_layout(int M, int N, int K, InputGradLayout* best) {
  const int* resident;
  if (int rc = input_grad_resident(&resident)) return rc;
  const int steps = div_up(N, 64);
  double least = 1e30;
  for (size_t i = 0; i < std::size(kInputGradLayouts); ++i) {
    const InputGradLayout l = kInputGradLayouts[i];
    if (l.slices > steps || resident[i] <= 0) continue;
    const long long tiles = (long long)div_up(M, 128 * l.cg) * div_up(K, 128 * l.cg);
    const double rounds = div_up(tiles, resident[i]);
    const double us = l.slices == 1 ? rounds * steps * 0.42 + 4 : rounds * (div_up(steps, l.slices) * 0.42 + 10.5);
    if (us < least) { least = us; *best = l; }
  }
  return WB200_OK;
}

template <int CG>
int launch_input_grad(const CUtensorMap& map, const CUtensorMap& codes, wb::InputGradParams p, int sms, cudaStream_t stream) {
  using Cfg = wb::InputGradCfg<CG>;
  p.tiles_m = div_up(p.M, Cfg::BM * CG);
  p.tiles_k = div_up(p.K, Cfg::TILE_K);
  p.group_k = std::min(8, p.tiles_k);
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  if (int rc = input_grad_config<CG>(p.slices, stream, &cfg, attr)) return rc;
  const long long tiles = (long long)p.tiles_m * p.tiles_k;
  cfg.gridDim.x = unsigned((p.slices > 1 ? tiles : std::min<long long>(tiles, sms / CG)) * CG * p.slices);
  WB_HOST_CUDA(cudaLaunchKernelEx(&cfg, wb::input_grad_kernel<CG>, map, codes, p));
  return WB200_OK;
}

// ------------------------------------------------------------------------------------------
// router
// ------------------------------------------------------------------------------------------
int router_ctas(int rows) { return rows <= wb::kRouterOneCta ? 1 : std::min(wb::kRouterMaxCtas, div_up(rows, wb::kRouterWarps)); }

int check_router(const char* what, int rows, int E, int top_k, int dtype, const void* logits, long long ld) {
  if (rows <= 0 || E <= 0 || top_k <= 0) return fail(WB200_ERR_INVALID_ARG, "%s: rows = %d, experts = %d, top_k = %d", what, rows, E, top_k);
  if (E > wb::kRouterMaxExperts) return fail(WB200_ERR_UNSUPPORTED, "%s: at most %d experts (got %d)", what, wb::kRouterMaxExperts, E);
  if (rows > 1 << 30 || (long long)rows * top_k > 0x7fffffffll) return fail(WB200_ERR_UNSUPPORTED, "%s: %d rows of %d choices in one call", what, rows, top_k);
  if (dtype != WB200_F32 && dtype != WB200_BF16) return fail(WB200_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  if (!logits) return fail(WB200_ERR_INVALID_ARG, "%s: null pointer", what);
  if (ld < E && rows > 1) return fail(WB200_ERR_INVALID_ARG, "%s: row pitch %lld is smaller than %d experts", what, ld, E);
  if (!aligned_to(logits, dtype == WB200_F32 ? 4 : 2)) return fail(WB200_ERR_ALIGNMENT, "%s: logits are not aligned to their element size", what);
  return WB200_OK;
}

// Lanes may load their experts (1, 2, 4 or 8 neighbours) as one piece.
int router_vec(const void* rows, long long ld, int E, int dtype) {
  const int per_lane = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : 8;
  return aligned_to(rows, 16) && ld * (dtype == WB200_F32 ? 4 : 2) % 16 == 0 && E % per_lane == 0;
}

#define WB_BY_EXPERTS(KERNEL, T, E)                                                                          \
  ((E) <= 32 ? KERNEL<T, 1> : (E) <= 64 ? KERNEL<T, 2> : (E) <= 128 ? KERNEL<T, 4> : KERNEL<T, 8>)

template <typename T, bool VEC, int SLOTS>
cudaError_t launch_combine_slots(const void* g, long long ldg, const void* y, long long ldy, const int* row_of, int tokens, int top_k, int cols,
                                float* g_weight, cudaStream_t s) {
  return launch(wb::combine_grad_kernel<T, VEC, SLOTS>, dim3(tokens), 128, 0, s, static_cast<const T*>(g), ldg, static_cast<const T*>(y), ldy, row_of,
                top_k, cols, g_weight);
}
template <typename T, bool VEC>
cudaError_t launch_combine_grad(const void* g, long long ldg, const void* y, long long ldy, const int* row_of, int tokens, int top_k, int cols,
                                float* g_weight, cudaStream_t s) {
  return top_k <= 2 ? launch_combine_slots<T, VEC, 2>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s)
                    : launch_combine_slots<T, VEC, 4>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s);
}

}  // namespace

namespace wbhost {
cudaError_t combine_tokens(const void* y, long long ldy, const int* row_of, const float* weight, int tokens, int top_k, int cols, void* out, long long ldo,
                           cudaStream_t stream) {
  auto kernel = top_k <= 2 ? wb::combine_token_kernel<2> : top_k <= 4 ? wb::combine_token_kernel<4> : wb::combine_token_kernel<8>;
  return launch(kernel, dim3(tokens), 128, 0, stream, static_cast<const __nv_bfloat16*>(y), ldy, row_of, weight, top_k, cols, static_cast<__nv_bfloat16*>(out), ldo);
}

cudaError_t adapt_check_record(unsigned long long (&record)[3], bool reset) {
#ifdef WB200_CHECKS
  cudaError_t e = cudaMemcpyFromSymbol(record, wb::g_check_record, sizeof(record));
  const unsigned long long zero[3] = {};
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(wb::g_check_record, zero, sizeof(zero));
  return e;
#else
  record[0] = record[1] = record[2] = 0;
  (void)reset;
  return cudaSuccess;
#endif
}
}  // namespace wbhost

extern "C" {

// One f32 a rank and row; callers that write f32 are asked for half as much again, of which nothing is used (the size that they know).
size_t wb200_adapters_hidden_bytes(int rows, int rank, int dtype) {
  if (rows <= 0 || rank <= 0) return 0;
  return size_t(rows) * (dtype == WB200_F32 ? 6 : 4) * rank_pad(rank);
}

int wb200_adapters_forward(int rows, int K, int N, int rank, int num_adapters, const void* x, long long ldx, const void* a, const void* b,
                           const void* ids, int ids_are_int64, const float* scale, const void* y, long long ldy, void* out, long long ldo, int dtype,
                           void* hidden, size_t hidden_bytes, void* stream) {
  if (int rc = check_adapters("adapters", rows, K, N, rank, num_adapters)) return rc;
  if (!x || !a || !b || !ids || !y || !out || !hidden) return fail(WB200_ERR_INVALID_ARG, "adapters: null pointer");
  if (dtype != WB200_F32 && dtype != WB200_BF16) return fail(WB200_ERR_INVALID_ARG, "adapters: unknown output dtype %d", dtype);
  if (rows > 1 && (ldx < K || ldy < N || ldo < N)) return fail(WB200_ERR_INVALID_ARG, "adapters: a row pitch is smaller than a row");
  if (ldy >= 1 << 24 || ldo >= 1 << 24) return fail(WB200_ERR_UNSUPPORTED, "adapters: a row pitch of 2^24 elements or more");
  if (!aligned_to(x, 2) || !aligned_to(a, 2) || !aligned_to(b, 2) || !aligned_to(y, dtype == WB200_F32 ? 4 : 2) || !aligned_to(out, dtype == WB200_F32 ? 4 : 2) ||
      !aligned_to(ids, ids_are_int64 ? 8 : 4) || !aligned_to(scale, 4) || !aligned_to(hidden, 16))
    return fail(WB200_ERR_ALIGNMENT, "adapters: a tensor is not aligned to its element size, or hidden not to 16 bytes");
  const size_t need = wb200_adapters_hidden_bytes(rows, rank, dtype);
  if (hidden_bytes < need) return fail(WB200_ERR_WORKSPACE, "adapters: hidden of %zu bytes needed (got %zu)", need, hidden_bytes);
  int *status = nullptr, sms = 0;
  if (int rc = wbhost::device(&sms, &status)) return rc;
  const AdapterCall c{{ids, ids_are_int64 != 0}, rows, rank, rank_pad(rank), num_adapters, static_cast<cudaStream_t>(stream), status, sms};
  auto* h = static_cast<float*>(hidden);
  if (int rc = run_shrink(c, static_cast<const __nv_bfloat16*>(x), ldx, K, static_cast<const __nv_bfloat16*>(a), false, scale, h)) return rc;
  return run_expand(c, static_cast<const __nv_bfloat16*>(b), false, h, y, ldy, out, ldo, dtype == WB200_F32, N);
}

size_t wb200_adapters_backward_workspace_bytes(int rows, int N, int rank) {
  if (rows <= 0 || N <= 0 || rank <= 0) return 0;
  const size_t hidden = (wb200_adapters_hidden_bytes(rows, rank, WB200_BF16) + 255) / 256 * 256;
  return hidden + (N % 8 ? size_t(rows) * ((N + 7) / 8 * 8) * 2 : 0);  // and a copy of g whose rows start on 16 bytes
}

int wb200_adapters_backward(int rows, int K, int N, int rank, int num_adapters, const void* x, long long ldx, const void* a, const void* b,
                            const void* ids, int ids_are_int64, const float* scale, const void* g, long long ldg, const void* hidden,
                            size_t hidden_bytes, void* dx, long long ldd, int accumulate_dx, void* da, void* db, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = check_adapters("adapters backward", rows, K, N, rank, num_adapters)) return rc;
  if (num_adapters > 65535) return fail(WB200_ERR_UNSUPPORTED, "adapters backward: at most 65535 adapters (got %d)", num_adapters);
  if (!dx && !da && !db) return fail(WB200_ERR_INVALID_ARG, "adapters backward: no gradient is asked for");
  if (!ids || !g || !workspace || ((dx || da) && !b) || (dx && !a) || (da && !x) || (db && !hidden))
    return fail(WB200_ERR_INVALID_ARG, "adapters backward: null pointer");
  if (rows > 1 && (ldg < N || (da && ldx < K) || (dx && ldd < K))) return fail(WB200_ERR_INVALID_ARG, "adapters backward: a row pitch is smaller than a row");
  if (ldd >= 1 << 24) return fail(WB200_ERR_UNSUPPORTED, "adapters backward: a row pitch of 2^24 elements or more");
  if (!aligned_to(x, 2) || !aligned_to(a, 2) || !aligned_to(b, 2) || !aligned_to(g, 2) || !aligned_to(dx, 2) || !aligned_to(da, 2) || !aligned_to(db, 2) ||
      !aligned_to(ids, ids_are_int64 ? 8 : 4) || !aligned_to(scale, 4) || !aligned_to(hidden, 16) || !aligned_to(workspace, 16))
    return fail(WB200_ERR_ALIGNMENT, "adapters backward: a tensor is not aligned to its element size, or hidden or the workspace not to 16 bytes");
  const size_t ws_need = wb200_adapters_backward_workspace_bytes(rows, N, rank);
  if (workspace_bytes < ws_need) return fail(WB200_ERR_WORKSPACE, "adapters backward: workspace of %zu bytes needed (got %zu)", ws_need, workspace_bytes);
  const size_t need = wb200_adapters_hidden_bytes(rows, rank, WB200_BF16);
  if (db && hidden_bytes < need) return fail(WB200_ERR_WORKSPACE, "adapters backward: hidden of %zu bytes needed (got %zu)", need, hidden_bytes);
  int *status = nullptr, sms = 0;
  if (int rc = wbhost::device(&sms, &status)) return rc;
  const AdapterCall c{{ids, ids_are_int64 != 0}, rows, rank, rank_pad(rank), num_adapters, static_cast<cudaStream_t>(stream), status, sms};
  const auto* gp = static_cast<const __nv_bfloat16*>(g);
  if (N % 8) {
    auto* copy = reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(workspace) + (need + 255) / 256 * 256);
    const int pitch = (N + 7) / 8 * 8;
    WB_HOST_CUDA(launch(wb::adapter_align_kernel, dim3(std::min(148 * 8, div_up((long long)rows * pitch / 8, 256))), 256, 0, c.stream, gp, ldg, rows, N, copy, pitch));
    gp = copy;
    ldg = pitch;
  }
  auto* u = static_cast<float*>(workspace);
  if (dx || da)
    if (int rc = run_shrink(c, gp, ldg, N, static_cast<const __nv_bfloat16*>(b), true, scale, u)) return rc;
  if (dx)
    if (int rc = run_expand(c, static_cast<const __nv_bfloat16*>(a), true, u, accumulate_dx ? dx : nullptr, ldd, dx, ldd, false, K)) return rc;
  if (da || db) {
    wb::OuterSide for_b = {gp, static_cast<const float*>(hidden), static_cast<__nv_bfloat16*>(db), ldg, N, 0, 0, 0};
    wb::OuterSide for_a = {static_cast<const __nv_bfloat16*>(x), u, static_cast<__nv_bfloat16*>(da), ldx, K, 0, 0, 1};
    return run_outer(c, for_b, for_a);
  }
  return WB200_OK;
}

int wb200_mxfp4_input_grad(int M, int N, int K, const void* g, long long ldg, const void* b, const void* b_scale, long long b_scale_stride, void* dx,
                           long long ldd, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0) return fail(WB200_ERR_INVALID_ARG, "input_grad: M, N, K must be positive (got %d, %d, %d)", M, N, K);
  if (K % 32) return fail(WB200_ERR_INVALID_ARG, "input_grad: K = %d is not a multiple of the scale group size 32", K);
  if (!g || !b || !b_scale || !dx) return fail(WB200_ERR_INVALID_ARG, "input_grad: null tensor pointer");
  if (M > 1 && (ldg < N || ldd < K)) return fail(WB200_ERR_INVALID_ARG, "input_grad: a row pitch is smaller than a row");
  if (N > 1 && b_scale_stride < K / 32) return fail(WB200_ERR_INVALID_ARG, "input_grad: the pitch of the scales is smaller than a row");
  if (M == 1) { ldg = (N + 7) / 8 * 8; ldd = K; }
  if (!aligned_to(g, 16) || ldg % 8 || !aligned_to(b, 16) || !aligned_to(dx, 16) || ldd % 8)
    return fail(WB200_ERR_ALIGNMENT, "input_grad: rows of g and dx and the codes must be 16-byte aligned");
  int sms = 0;
  wb::InputGradParams p;
  if (int rc = wbhost::device(&sms, &p.status)) return rc;
  p.scales = static_cast<const uint8_t*>(b_scale);
  p.dx = static_cast<__nv_bfloat16*>(dx);
  p.ld_scales = b_scale_stride; p.ldd = ldd;
  p.M = M; p.N = N; p.K = K;
  p.scale_words = aligned_to(b_scale, 4) && b_scale_stride % 4 == 0 && K % 128 == 0;
  CUtensorMap map, codes;
  if (int rc = wbhost::tensor_map(&codes, b, K / 2, N, K / 2, 64, 64, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
  if (int rc = wbhost::tensor_map(&map, g, N, M, (unsigned long long)ldg * 2, 64, 128, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  InputGradLayout layout{2, 1};
  if (int rc = input_grad_layout(M, N, K, &layout)) return rc;
  p.slices = layout.slices;
  return layout.cg == 2 ? launch_input_grad<2>(map, codes, p, sms, s) : launch_input_grad<1>(map, codes, p, sms, s);
}

size_t wb200_router_workspace_bytes(int rows, int num_experts) {
  if (rows <= 0 || num_experts <= 0) return 0;
  return size_t(router_ctas(rows)) * (2 * num_experts + 1) * 4;
}

int wb200_router(int rows, int num_experts, int top_k, const void* logits, int dtype, long long ld, const void* mask, const void* given_ids,
                 int given_are_int64, int renormalize, float* weight, int* ids, int* counts, float* unit, float* loss, void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (int rc = check_router("router", rows, num_experts, top_k, dtype, logits, ld)) return rc;
  if (!given_ids && (top_k > num_experts || top_k > wb::kRouterMaxTopK))
    return fail(WB200_ERR_INVALID_ARG, "router: top_k = %d with %d experts (at most %d)", top_k, num_experts, wb::kRouterMaxTopK);
  if ((!given_ids && (!weight || !ids)) || !counts || !unit || !loss || !workspace) return fail(WB200_ERR_INVALID_ARG, "router: null pointer");
  const size_t need = wb200_router_workspace_bytes(rows, num_experts);
  if (workspace_bytes < need) return fail(WB200_ERR_WORKSPACE, "router: workspace of %zu bytes needed (got %zu)", need, workspace_bytes);
  if (!aligned_to(workspace, 4)) return fail(WB200_ERR_ALIGNMENT, "router: the workspace must be 4-byte aligned");
  if (!words_aligned({weight, ids, counts, unit, loss}) || !aligned_to(given_ids, given_are_int64 ? 8 : 4))
    return fail(WB200_ERR_ALIGNMENT, "router: a tensor is not aligned to its element size");
  if (int rc = wbhost::device(nullptr, nullptr)) return rc;
  wb::RouterParams p;
  p.logits = logits; p.mask = static_cast<const uint8_t*>(mask); p.given = given_ids; p.ld = ld;
  p.rows = rows; p.E = num_experts; p.top_k = top_k; p.renormalize = renormalize; p.given_i64 = given_are_int64;
  p.weight = weight; p.ids = ids; p.counts = counts; p.unit = unit; p.loss = loss;
  p.vec = router_vec(logits, ld, num_experts, dtype);
  const int ctas = router_ctas(rows);
  p.part_p = static_cast<float*>(workspace);
  p.part_n = reinterpret_cast<int*>(p.part_p + size_t(ctas) * num_experts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  void (*kernel)(wb::RouterParams) = dtype == WB200_F32 ? WB_BY_EXPERTS(wb::router_kernel, float, num_experts) : WB_BY_EXPERTS(wb::router_kernel, __nv_bfloat16, num_experts);
  WB_HOST_CUDA(launch(kernel, dim3(ctas), wb::kRouterWarps * 32, 0, s, p));
  if (ctas > 1) WB_HOST_CUDA(launch_clusters(wb::router_finish_kernel, dim3(div_up(num_experts, 32)), 1024, 0, s, p, ctas));
  return WB200_OK;
}

int wb200_router_grad(int rows, int num_experts, int top_k, const void* logits, int dtype, long long ld, const void* mask, const int* ids,
                      const float* g_weight, const float* g_loss, int renormalize, const int* counts, const float* unit, void* g_logits,
                      long long ldg, void* stream) {
  if (int rc = check_router("router gradient", rows, num_experts, top_k, dtype, logits, ld)) return rc;
  if (!counts || !unit || !g_logits || (g_weight && !ids)) return fail(WB200_ERR_INVALID_ARG, "router gradient: null pointer");
  if (g_weight && (top_k > num_experts || top_k > wb::kRouterMaxTopK))
    return fail(WB200_ERR_INVALID_ARG, "router gradient: top_k = %d with %d experts (at most %d)", top_k, num_experts, wb::kRouterMaxTopK);
  if (rows > 1 && ldg < num_experts) return fail(WB200_ERR_INVALID_ARG, "router gradient: row pitch %lld is smaller than %d experts", ldg, num_experts);
  if (!words_aligned({ids, g_weight, g_loss, counts, unit}) || !aligned_to(g_logits, dtype == WB200_F32 ? 4 : 2))
    return fail(WB200_ERR_ALIGNMENT, "router gradient: a tensor is not aligned to its element size");
  if (int rc = wbhost::device(nullptr, nullptr)) return rc;
  wb::RouterGradParams p;
  p.logits = logits; p.mask = static_cast<const uint8_t*>(mask); p.ids = ids; p.g_weight = g_weight; p.g_loss = g_loss; p.counts = counts;
  p.unit = unit; p.g_logits = g_logits; p.ld = ld; p.ldg = ldg;
  p.rows = rows; p.E = num_experts; p.top_k = top_k; p.renormalize = renormalize;
  p.vec = router_vec(logits, ld, num_experts, dtype) && router_vec(g_logits, ldg, num_experts, dtype);
  void (*kernel)(wb::RouterGradParams) =
      dtype == WB200_F32 ? WB_BY_EXPERTS(wb::router_grad_kernel, float, num_experts) : WB_BY_EXPERTS(wb::router_grad_kernel, __nv_bfloat16, num_experts);
  WB_HOST_CUDA(launch(kernel, dim3(std::min(1184, div_up(rows, wb::kRouterWarps))), wb::kRouterWarps * 32, 0, static_cast<cudaStream_t>(stream), p));
  return WB200_OK;
}

int wb200_moe_combine_grad(const void* g, long long ldg, const void* y, long long ldy, int dtype, const int* row_of, int tokens, int top_k, int cols,
                           float* g_weight, void* stream) {
  if (tokens <= 0 || top_k <= 0 || cols <= 0)
    return fail(WB200_ERR_INVALID_ARG, "moe_combine_grad: tokens = %d, top_k = %d, cols = %d", tokens, top_k, cols);
  if (!g || !y || !row_of || !g_weight) return fail(WB200_ERR_INVALID_ARG, "moe_combine_grad: null pointer");
  if (dtype != WB200_F32 && dtype != WB200_BF16) return fail(WB200_ERR_INVALID_ARG, "moe_combine_grad: unknown dtype %d", dtype);
  if (ldy < cols || (tokens > 1 && ldg < cols)) return fail(WB200_ERR_INVALID_ARG, "moe_combine_grad: a row pitch is smaller than cols = %d", cols);
  if (!words_aligned({row_of, g_weight}) || !aligned_to(g, dtype == WB200_F32 ? 4 : 2) || !aligned_to(y, dtype == WB200_F32 ? 4 : 2))
    return fail(WB200_ERR_ALIGNMENT, "moe_combine_grad: a tensor is not aligned to its element size");
  if (int rc = wbhost::device(nullptr, nullptr)) return rc;
  const size_t esz = dtype == WB200_F32 ? 4 : 2;
  const bool vec = cols % 8 == 0 && aligned_to(g, 16) && aligned_to(y, 16) && ldg * esz % 16 == 0 && ldy * esz % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == WB200_F32)
    WB_HOST_CUDA(vec ? launch_combine_grad<float, true>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s)
                     : launch_combine_grad<float, false>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s));
  else
    WB_HOST_CUDA(vec ? launch_combine_grad<__nv_bfloat16, true>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s)
                     : launch_combine_grad<__nv_bfloat16, false>(g, ldg, y, ldy, row_of, tokens, top_k, cols, g_weight, s));
  return WB200_OK;
}

}  // extern "C"
