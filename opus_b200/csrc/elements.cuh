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

// Two 16-bit elements in a word, low half first.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// V elements of T in one access of at most 16 bytes (V * sizeof(T) a power of two), kept as words: taking 16-bit
// elements apart one by one costs several instructions each.
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  uint32_t w[V / 2];
  __device__ __forceinline__ void get(float (&r)[V]) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = unpack2<T>(w[i]);
      r[2 * i] = f.x, r[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ void set(const float (&r)[V]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2<T>(r[2 * i], r[2 * i + 1]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = 0u;
  }
};
template <int V>
struct alignas(V * 4) Vec<float, V> {
  float w[V];
  __device__ __forceinline__ void get(float (&r)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = w[i];
  }
  __device__ __forceinline__ void set(const float (&r)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = r[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 0.f;
  }
};
template <typename T>
struct Vec<T, 1> {
  T w;
  __device__ __forceinline__ void get(float (&r)[1]) const { r[0] = to_f32(w); }
  __device__ __forceinline__ void set(const float (&r)[1]) { w = from_f32<T>(r[0]); }
  __device__ __forceinline__ void zero() { w = from_f32<T>(0.f); }
};
template <>
struct Vec<float, 1> {
  float w;
  __device__ __forceinline__ void get(float (&r)[1]) const { r[0] = w; }
  __device__ __forceinline__ void set(const float (&r)[1]) { w = r[0]; }
  __device__ __forceinline__ void zero() { w = 0.f; }
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&r)[V]) {
  const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(p);
  x.get(r);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&r)[V]) {
  Vec<T, V> x;
  x.set(r);
  *reinterpret_cast<Vec<T, V>*>(p) = x;
}

// Arithmetic on vectors of f32; Pairs: two elements to an instruction, for kernels that are bound by the instructions
// they issue and have registers to spare (pairs lie in neighbouring ones).  The roundings are those of one by one.
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
// (a, b) = (a x0 + y0, b x1 + y1)
__device__ __forceinline__ void fma2(float& a, float& b, float x0, float x1, float y0, float y1) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}
// (a, b) += (x0 y0, x1 y1)
__device__ __forceinline__ void mac2(float& a, float& b, float x0, float x1, float y0, float y1) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}
// r += s, r *= s, r += a, r *= a, r = r a + b, r = r s + b, r += a b, elementwise
template <bool Pairs, int V>
__device__ __forceinline__ void vadd(float (&r)[V], float s) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] += s;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) add2(r[i], r[i + 1], s, s);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vmul(float (&r)[V], float s) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] *= s;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) mul2(r[i], r[i + 1], s, s);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vadd(float (&r)[V], const float (&a)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] += a[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) add2(r[i], r[i + 1], a[i], a[i + 1]);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vmul(float (&r)[V], const float (&a)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] *= a[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) mul2(r[i], r[i + 1], a[i], a[i + 1]);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vfma(float (&r)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = fmaf(r[i], a[i], b[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) fma2(r[i], r[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vfma(float (&r)[V], float s, const float (&b)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = fmaf(r[i], s, b[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) fma2(r[i], r[i + 1], s, s, b[i], b[i + 1]);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vmac(float (&r)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = fmaf(a[i], b[i], r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) mac2(r[i], r[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
  }
}
// (s0, s1) += the vector's elements (products) in two chains
template <bool Pairs, int V>
__device__ __forceinline__ void vsum(float (&s)[2], const float (&a)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i & 1] += a[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) add2(s[0], s[1], a[i], a[i + 1]);
  }
}
template <bool Pairs, int V>
__device__ __forceinline__ void vdot(float (&s)[2], const float (&a)[V], const float (&b)[V]) {
  if constexpr (!Pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i & 1] = fmaf(a[i], b[i], s[i & 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) mac2(s[0], s[1], a[i], a[i + 1], b[i], b[i + 1]);
  }
}

// One element into an array whose type is known at run time (the parameters' gradients).
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
