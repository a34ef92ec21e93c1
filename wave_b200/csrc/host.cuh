// What the library's translation units share on the host: the error message of the calling thread, the device's set-up and the
// tensor-map cache (defined in api.cu, not exported).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/wave_b200.h"

#define WB_HIDDEN __attribute__((visibility("hidden")))

namespace wbhost {

constexpr int kMaxDevices = 64;

WB_HIDDEN int fail(int code, const char* fmt, ...);             // keeps the message, returns code
WB_HIDDEN int device(int* sm_count, int** status);              // of the current device; status may be null
// A 2-D tensor map: d0 x d1 elements (d0 contiguous), rows `stride` bytes apart, boxes of box0 x box1.
WB_HIDDEN int tensor_map(CUtensorMap* map, const void* base, unsigned long long d0, unsigned long long d1, unsigned long long stride,
                         unsigned box0, unsigned box1, CUtensorMapDataType dtype, CUtensorMapSwizzle swizzle,
                         CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_NONE);
// moe_combine for bf16 rows that start on 16 bytes, at most 8 pairs a token (adapt.cu).
WB_HIDDEN cudaError_t combine_tokens(const void* y, long long ldy, const int* row_of, const float* weight, int tokens, int top_k, int cols, void* out,
                                     long long ldo, cudaStream_t stream);
// The debug-checked build keeps a record per translation unit.
WB_HIDDEN cudaError_t adapt_check_record(unsigned long long (&record)[3], bool reset);

}  // namespace wbhost

#define WB_HOST_CUDA(...)                                                                                              \
  do {                                                                                                                 \
    cudaError_t e__ = (__VA_ARGS__);                                                                                   \
    if (e__ != cudaSuccess)                                                                                            \
      return wbhost::fail(WB200_ERR_CUDA, "%s failed: %s (%s:%d)", #__VA_ARGS__, cudaGetErrorString(e__), __FILE__, __LINE__); \
  } while (0)
