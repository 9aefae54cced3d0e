// nsfps_feature.cuh -- helpers shared by the feature operators
// (nsfps_rows.cu, nsfps_select.cu, nsfps_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

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

// What a launch asks of the current device, once per device (up to 64).
inline int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

inline int sm_count() {
  static std::atomic<int> known[64];
  const int dev = current_device();
  int sms = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms = 148;
  if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// More than 48 KB of shared memory a CTA, the static included, has to be asked
// for, per kernel (hence the template) and device.
template <auto Kernel>
cudaError_t opt_in(uint32_t smem) {
  if (smem <= 40u << 10) return cudaSuccess;
  static std::atomic<uint64_t> asked;
  const int dev = current_device();
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (asked.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t err =
      cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return err;
}

// Launches a kernel that begins with after_previous() behind the one before it
// in the stream: its CTAs are set up while that one's last results go out
// (attention over a scan 200 -> 178 us; letting them in earlier, beside CTAs
// that still run, 183).
template <class... P, class... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t smem,
                        cudaStream_t st, const A &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// First in every kernel that launch_next starts, by all threads: the kernels
// before have ended and what they wrote is there.
__device__ __forceinline__ void after_previous() { cudaGridDependencySynchronize(); }

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

}  // namespace nsfps
