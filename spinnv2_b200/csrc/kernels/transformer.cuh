// Shared helpers of the decoder-layer operators (norm_i8.cu, linear_i8.cu,
// cross_attention.cu): element types and argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "spkv2_transformer.h"

#include "common.cuh"

namespace spkv2 {
namespace xf {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

inline int elem_bytes(int32_t dtype) {
  return dtype == SPKV2_DTYPE_FP32 ? 4 : (dtype == SPKV2_DTYPE_FP16 || dtype == SPKV2_CUDA_DTYPE_BF16) ? 2 : 0;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether output rows `stride` apart would overlap.  Inputs may (stride 0:
// one row for all).
inline bool overlaps(int64_t stride, int64_t rows, int64_t width) { return rows > 1 ? stride < width : stride < 0; }

// Whether every pointer given (NULL counts as given) is a multiple of `bytes`.
template <class... P>
inline bool on_bytes(uintptr_t bytes, const P *...p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0;
}

// Calls fn(T{}) for the element type of `dtype`, which the caller has checked.
template <class F>
inline int by_type(int32_t dtype, F &&fn) {
  switch (dtype) {
    case SPKV2_DTYPE_FP32: return fn(float{});
    case SPKV2_DTYPE_FP16: return fn(__half{});
    case SPKV2_CUDA_DTYPE_BF16: return fn(__nv_bfloat16{});
    default: return SPKV2_ERR_UNSUPPORTED;
  }
}

// The current device's SMs; 148 where the runtime cannot be asked.
inline int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return 148;
    return v;
  }();
  return n;
}

// Lets KERN use `bytes` of dynamic shared memory on the current device; asked
// of the driver once for each device.
template <auto KERN>
inline int allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SPKV2_ERR_NO_DEVICE;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  const cudaError_t err = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return cuda_status(err);
}

// Reads and clears the status word (a device variable) of a file's kernels on
// the current device, whose work has ended.
template <class Word>
inline int take_status(Word &word, int *code) {
  *code = 0;
  cudaError_t err = cudaMemcpyFromSymbol(code, word, sizeof(int));
  const int zero = 0;
  if (err == cudaSuccess && *code) err = cudaMemcpyToSymbol(word, &zero, sizeof(int));
  return cuda_status(err);
}

}  // namespace xf

// The status words of the kernels that wait with a limit.
int linear_status(int *code);
int cross_tc_status(int *code);
int cross_step_status(int *code);

}  // namespace spkv2
