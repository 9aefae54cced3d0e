// nsfps_feature.cuh -- helpers shared by the feature operators
// (nsfps_rows.cu, nsfps_select.cu, nsfps_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nsfps_internal.cuh"
#include "nsfps_kernels.h"

namespace nsfps {

#define NSFPS_FEATURE_CUDA(call)                                                   \
  do {                                                                             \
    cudaError_t e_ = (call);                                                       \
    if (e_ != cudaSuccess)                                                         \
      return set_error(NSFPS_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_)); \
  } while (0)

// Hands out 256-byte aligned pieces of the caller's scratch (base nullptr: only
// counts).
struct WorkCarver {
  char *base;
  uint64_t off = 0;
  explicit WorkCarver(void *p) : base((char *)p) {}
  template <class T>
  T *take(uint64_t count) {
    T *p = base ? (T *)(base + off) : nullptr;
    off += (count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

inline int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Scratch of run_sort_pairs over n pairs (its second buffers included).
struct SortScratch {
  uint32_t *keys0, *vals0, *keys1, *vals1, *hist, *partial;
  void carve(WorkCarver &w, uint32_t n) {
    const uint64_t h = 256ull * radix_tiles(n) + 1;
    keys0 = w.take<uint32_t>(n);
    vals0 = w.take<uint32_t>(n);
    keys1 = w.take<uint32_t>(n);
    vals1 = w.take<uint32_t>(n);
    hist = w.take<uint32_t>(h);
    partial = w.take<uint32_t>(h / 4096 + 3);
  }
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// First position in the ascending keys[0 .. n) whose key is >= v.
__device__ __forceinline__ uint32_t lower_bound(const uint32_t *__restrict__ keys, uint32_t n,
                                                uint32_t v) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

}  // namespace nsfps
