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

// Untiled bulk copy global -> shared: both 16-byte aligned, bytes a multiple of 16.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

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

// Two 16-bit values of a word (the first in its low half), widened; and back, rounded.
template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack16<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight consecutive values as they lie in memory (16 bytes, 32 for fp32), in registers.
template <typename T>
struct Raw8 {
  static constexpr int WORDS = sizeof(T) * 2;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i / 4];
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack16<T>(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack16<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};

}  // namespace actune
