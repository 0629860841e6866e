// Element types of the training operators: 16-byte loads and stores of f32,
// bf16 and f16 as floats, and single elements of a type chosen at run time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/emeans_b200.h"

namespace eb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// Element i of an array of a float type known at run time.
__device__ __forceinline__ float load_any(const void* p, int dtype, size_t i) {
  if (dtype == EB_F32) return static_cast<const float*>(p)[i];
  if (dtype == EB_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, size_t i, float v) {
  if (dtype == EB_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == EB_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// V elements as loaded (V * sizeof(T) is 16 bytes, or V is 1).
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
};

}  // namespace eb
