// Element conversions and 16-byte row pieces shared by the 8-bit and routing
// kernels.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace g2q {
namespace rows {

template <typename S>
__device__ __forceinline__ float to_f(S v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <typename S>
__device__ __forceinline__ S of_f(float v);
template <>
__device__ __forceinline__ float of_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 of_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half of_f<__half>(float v) { return __float2half_rn(v); }

static inline int elem_bytes(int dtype) {
  return dtype == G2Q_DTYPE_F32 ? 4 : (dtype == G2Q_DTYPE_BF16 || dtype == G2Q_DTYPE_F16) ? 2 : 0;
}

static inline bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0;
}

}  // namespace rows
}  // namespace g2q
