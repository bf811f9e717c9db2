// Element access of the training-step kernels: values of bf16, f16 or f32 as
// f32 in registers, in vectors of up to 16 bytes, each rounded once on the
// way out (round to nearest even).
#pragma once

#include <cuda_fp16.h>

#include "opus_common.cuh"

namespace opus {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// V elements of T in one access of at most 16 bytes (V * sizeof(T) a power of two).
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&r)[V]) {
  const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = to_f32(x.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&r)[V]) {
  Vec<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(r[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = x;
}

// One element of an array whose type is known at run time (parameters: read once per block or row).
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == OPUS_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == OPUS_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == OPUS_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == OPUS_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__host__ __device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == OPUS_DTYPE_F32 ? 4 : 2; }
__host__ __device__ __forceinline__ bool dtype_ok(int dtype) {
  return dtype == OPUS_DTYPE_BF16 || dtype == OPUS_DTYPE_F32 || dtype == OPUS_DTYPE_F16;
}

}  // namespace opus
