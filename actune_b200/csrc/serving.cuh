// Internal declarations of the serving operators (include/actune_b200_serving.h).
#pragma once

#include <cudaTypedefs.h>

#include "actune_b200.h"
#include "actune_b200_serving.h"
#include "common.cuh"
#include "kernels.cuh"

namespace actune {

// capi.cu: the current device's checks (ACTUNE_OK, or why it cannot run this library),
// its SM count, the driver's tensor-map encoder and the CUDA-error bookkeeping.
int serving_device(int* num_sms);
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();
int serving_status(cudaError_t e);

inline bool is_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive values as they lie in memory (16 bytes, 32 for fp32).
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = widen<T>(t[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    T* t = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = narrow<T>(v[i]);
  }
};

}  // namespace actune
