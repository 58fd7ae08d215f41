// Element types of the operators on device buffers: conversions to and from
// fp32 (one rounding to nearest), and the dispatch over FE_DTYPE_*.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/flowedge_b200.h"

namespace feb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
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

// body(T{}) for the element type of `dtype`
template <typename F>
int with_dtype(unsigned dtype, F body) {
  if (dtype == FE_DTYPE_F32) return body(float{});
  if (dtype == FE_DTYPE_BF16) return body(__nv_bfloat16{});
  return body(__half{});
}

}  // namespace feb
