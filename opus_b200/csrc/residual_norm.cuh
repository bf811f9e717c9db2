// Rows of the residual norm in registers: the parts that its forward and
// backward kernels share.
//
// A row of d elements is held by a group of `group` threads (a power of two up
// to 32, or whole warps), thread t holding the vectors t, t + group, ... of V
// elements each, NV of them at most.  A block holds `groups` rows at a time.
#pragma once

#include "elements.cuh"

namespace opus {

constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxWidth = 16384;

// Threads of a block at most, by the elements that a thread holds (norm_shape keeps to it).
constexpr int norm_threads(int V, int NV) { return V * NV >= 16 ? 1024 : 512; }

struct NormShape {
  int64_t rows;
  int64_t seq;  // rows that share a row of the gate (rows of a sample); `rows` for one gate
  int d;
  int group, groups;  // threads of a row, rows of a block
  int layer;          // LayerNorm (1) or RMS norm (0)
  float eps;
};

// Sums over the group of up to two values each, one after the other in a fixed
// order; the result is in every thread of the group.  `turn` alternates between
// calls, so that one barrier a call is enough.
struct GroupSum {
  float* buf;  // 2 * 2 * warps floats of shared memory
  int group, warps, warp, lane, first;
  int turn;

  __device__ GroupSum(float* shared, int group_) : buf(shared), group(group_), turn(0) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    warps = blockDim.x >> 5;
    first = (threadIdx.x / group) * (group >> 5);  // of the group's warps, when it has whole ones
  }
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    const int width = group < 32 ? group : 32;
#pragma unroll
    for (int i = 0; i < N; ++i)
      for (int o = width >> 1; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (group <= 32) return;
    float* b = buf + turn * 2 * warps;
    turn ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[i * warps + warp] = v[i];
    }
    __syncthreads();
    const int n = group >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
      for (int w = 0; w < n; ++w) s += b[i * warps + first + w];
      v[i] = s;
    }
  }
};

// mean (0 for an RMS norm) and 1 / sqrt(mean square about it + eps) of the row held in r.
template <int NV, int V>
__device__ __forceinline__ float2 row_stats(const float (&r)[NV][V], const NormShape& s, int t, GroupSum& sum) {
  float mean = 0.f;
  const float inv_d = 1.0f / static_cast<float>(s.d);
  if (s.layer) {
    float a[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) a[0] += r[k][i];  // zeros beyond the row
    sum(a);
    mean = a[0] * inv_d;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if ((k * s.group + t) * V >= s.d) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float c = r[k][i] - mean;
      q[0] = fmaf(c, c, q[0]);
    }
  }
  sum(q);
  return make_float2(mean, rsqrtf(q[0] * inv_d + s.eps));
}

// V neighbours of a parameter vector, or `other` where there is none.
template <int V>
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t at, float other, float (&r)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = p != nullptr ? load_any(p, dtype, at + i) : other;
}

int norm_shape(const char* what, const opus_residual_norm_args* a, bool vec, int V, NormShape* s, int* nv);
int check_norm(const char* what, const opus_residual_norm_args* a);

}  // namespace opus
