// Conversions and vector access shared by the kernels of the quantised linear layer.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "linear.hpp"

namespace imd {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements of T moved as one access (16 bytes or a single element).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// The value of a scale stored as `type`, element i.
__device__ __forceinline__ float load_scale(const void* p, int32_t type, int64_t i) {
  if (type == IMD_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == IMD_TYPE_F16) return to_float(static_cast<const __half*>(p)[i]);
  return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
}

}  // namespace imd
