// Residual norm, forward: the joint between two blocks in one pass.
//
//   z = y or N(y) w_post + b_post;  h = r x + g z;  n = N(h) w + b
//
// N(v) = v / sqrt(mean v^2 + eps), or (v - mean) / sqrt(var + eps) with the
// variance summed about the mean (two sums over the registers, so no
// cancellation).  n is the norm of the h that is stored: what the next block
// sees is the norm of the residual stream as the backward will read it.
//
// Bound: HBM bandwidth; x and y are read once, h and n written once, nothing
// else but 16 bytes of statistics a row.
#include "residual_norm.cuh"

namespace opus {

int check_norm(const char* what, const opus_residual_norm_args* a) {
  if (a == nullptr) return set_error(OPUS_ERR_INVALID, "%s: NULL arguments", what);
  if (a->rows < 0 || a->d < 1) return set_error(OPUS_ERR_INVALID, "%s: bad sizes rows=%lld d=%d", what, (long long)a->rows, a->d);
  if (a->d > kNormMaxWidth) return set_error(OPUS_ERR_UNSUPPORTED, "%s: d up to %d (got %d)", what, kNormMaxWidth, a->d);
  if (a->kind != 0 && a->kind != 1) return set_error(OPUS_ERR_INVALID, "%s: kind %d is neither 0 (RMS) nor 1 (layer)", what, a->kind);
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->y_dtype) || (a->x_dtype != a->y_dtype && a->x_dtype != OPUS_DTYPE_F32))
    return set_error(OPUS_ERR_UNSUPPORTED, "%s: x is of y's type (bf16, f16 or f32) or f32", what);
  if (a->post && a->y == nullptr && a->rows > 0) return set_error(OPUS_ERR_INVALID, "%s: a norm after the block needs y", what);
  if (!a->post && (a->post_weight || a->post_bias))
    return set_error(OPUS_ERR_INVALID, "%s: post_weight and post_bias belong to post", what);
  const void* p[5] = {a->weight, a->bias, a->post_weight, a->post_bias, a->gate};
  const int t[5] = {a->weight_dtype, a->bias_dtype, a->post_weight_dtype, a->post_bias_dtype, a->gate_dtype};
  for (int i = 0; i < 5; ++i) {
    if (p[i] == nullptr) continue;
    if (!dtype_ok(t[i])) return set_error(OPUS_ERR_UNSUPPORTED, "%s: a parameter is neither bf16, f16 nor f32", what);
    if (reinterpret_cast<uintptr_t>(p[i]) % dtype_bytes(t[i]) != 0)
      return set_error(OPUS_ERR_INVALID, "%s: a parameter is not aligned to its elements", what);
  }
  if (a->gate != nullptr) {
    if (a->y == nullptr && a->rows > 0) return set_error(OPUS_ERR_INVALID, "%s: a gate needs y", what);
    if (a->gate_rows < 1 || a->rows % a->gate_rows != 0)
      return set_error(OPUS_ERR_INVALID, "%s: %lld rows cannot share %lld gate rows evenly", what, (long long)a->rows,
                       (long long)a->gate_rows);
  }
  return OPUS_OK;
}

// The launch's shape for vectors of V elements: as few vectors a thread as keep a row within 512 threads
// (more warps of one row hide its loads better than more loads of one warp), up to 1024 for the widest rows.
int norm_shape(const char* what, const opus_residual_norm_args* a, bool vec, int V, NormShape* s, int* nv) {
  if (!vec) V = 1;
  const int full = (a->d + V - 1) / V;
  const int steps[3] = {V == 1 ? 4 : 1, V == 1 ? 16 : 2, V == 1 ? 16 : 4};
  int k = 0;
  while (k < 2 && (full + steps[k] - 1) / steps[k] > 512) ++k;
  if (V == 8 && k == 2) k = 1;
  *nv = steps[k];
  int need = (full + *nv - 1) / *nv;
  int group = 1;
  if (need <= 32) {
    while (group < need) group <<= 1;
  } else {
    group = (need + 31) / 32 * 32;
  }
  if (group > kNormMaxThreads) return set_error(OPUS_ERR_UNSUPPORTED, "%s: d = %d is too wide", what, a->d);
  s->rows = a->rows;
  s->seq = a->gate != nullptr && a->gate_rows > 0 ? a->rows / a->gate_rows : a->rows;
  if (s->seq < 1) s->seq = 1;
  s->d = a->d;
  s->group = group;
  s->groups = group >= 256 ? 1 : 256 / group;
  s->layer = a->kind;
  s->eps = a->eps;
  return OPUS_OK;
}

namespace {

template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(norm_threads(V, NV))
    residual_norm_kernel(const __grid_constant__ NormShape s,
                                     const __grid_constant__ opus_residual_norm_args a) {
  extern __shared__ float shared[];
  GroupSum sum(shared, s.group);
  const int t = threadIdx.x % s.group;
  const int64_t in_block = threadIdx.x / s.group;
  const TX* x = static_cast<const TX*>(a.x);
  const TY* y = static_cast<const TY*>(a.y);
  TX* hp = static_cast<TX*>(a.h);
  TY* np = static_cast<TY*>(a.n);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * s.groups; base < s.rows;
       base += static_cast<int64_t>(gridDim.x) * s.groups) {
    const int64_t row = base + in_block;
    const bool live = row < s.rows;
    float h[NV][V], z[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) h[k][i] = z[k][i] = 0.f;
      if (live && col < s.d) {
        load_vec<TX, V>(x + row * a.x_stride + col, h[k]);
        if (y != nullptr) load_vec<TY, V>(y + row * a.y_stride + col, z[k]);
      }
    }
    float2 ys = make_float2(0.f, 0.f);
    if (a.post) {
      ys = row_stats<NV, V>(z, s, t, sum);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (k * s.group + t) * V;
        if (col >= s.d) continue;
        float w[V], b[V];
        load_param<V>(a.post_weight, a.post_weight_dtype, col, 1.f, w);
        load_param<V>(a.post_bias, a.post_bias_dtype, col, 0.f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) z[k][i] = (z[k][i] - ys.x) * ys.y * w[i] + b[i];
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
      if (col >= s.d || !live) continue;
      if (y != nullptr) {
        float g[V];
        load_param<V>(a.gate, a.gate_dtype, row / s.seq * s.d + col, 1.f, g);
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = a.residual_scale * h[k][i] + g[i] * z[k][i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = a.residual_scale * h[k][i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) h[k][i] = to_f32(from_f32<TX>(h[k][i]));
      if (hp != nullptr) store_vec<TX, V>(hp + row * s.d + col, h[k]);
    }
    const float2 hs = row_stats<NV, V>(h, s, t, sum);
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
      if (col >= s.d) continue;
      float w[V], b[V];
      load_param<V>(a.weight, a.weight_dtype, col, 1.f, w);
      load_param<V>(a.bias, a.bias_dtype, col, 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) h[k][i] = (h[k][i] - hs.x) * hs.y * w[i] + b[i];
      store_vec<TY, V>(np + row * s.d + col, h[k]);
    }
    if (t == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(hs.x, hs.y, ys.x, ys.y);
  }
}

template <typename TX, typename TY, int V, int NV>
int launch(const NormShape& s, const opus_residual_norm_args& a, cudaStream_t st) {
  const int threads = (s.group * s.groups + 31) / 32 * 32;
  int64_t blocks = (s.rows + s.groups - 1) / s.groups;
  const int64_t most = static_cast<int64_t>(sm_count()) * (2048 / threads);
  if (blocks > most) blocks = most;
  residual_norm_kernel<TX, TY, V, NV><<<static_cast<unsigned>(blocks), threads, 4 * (threads / 32) * sizeof(float), st>>>(s, a);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename TX, typename TY>
int launch_by_width(const opus_residual_norm_args& a, bool vec, cudaStream_t st) {
  constexpr int V = 16 / sizeof(TX);
  NormShape s;
  int nv;
  const int rc = norm_shape("residual_norm", &a, vec, V, &s, &nv);
  if (rc) return rc;
  if (!vec) return nv == 4 ? launch<TX, TY, 1, 4>(s, a, st) : launch<TX, TY, 1, 16>(s, a, st);
  if (nv == 1) return launch<TX, TY, V, 1>(s, a, st);
  if (nv == 2) return launch<TX, TY, V, 2>(s, a, st);
  if constexpr (V == 4) return launch<TX, TY, V, 4>(s, a, st);
  return set_error(OPUS_ERR_UNSUPPORTED, "residual_norm: d = %d", a.d);
}

bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace opus

using namespace opus;

extern "C" int opus_residual_norm(const opus_residual_norm_args* args, void* stream) {
  int rc = check_norm("residual_norm", args);
  if (rc) return rc;
  opus_residual_norm_args a = *args;
  if (a.rows == 0) return OPUS_OK;
  if (!a.x || !a.n || !a.stats) return set_error(OPUS_ERR_INVALID, "residual_norm: NULL pointer");
  if (!a.h && (a.y || a.residual_scale != 1.0f))
    return set_error(OPUS_ERR_INVALID, "residual_norm: h is NULL, and differs from x");
  const int xb = dtype_bytes(a.x_dtype), yb = dtype_bytes(a.y_dtype);
  if (a.x_stride < a.d || (a.y && a.y_stride < a.d)) return set_error(OPUS_ERR_INVALID, "residual_norm: row stride < d");
  if (!on(a.x, xb) || !on(a.h, xb) || !on(a.y, yb) || !on(a.n, yb) || !on(a.stats, 16))
    return set_error(OPUS_ERR_INVALID, "residual_norm: a pointer is not aligned to its elements");
  const int V = 16 / xb;
  const bool vec = a.d % V == 0 && a.x_stride % V == 0 && on(a.x, 16) && on(a.h, 16) && on(a.n, V * yb) &&
                   (!a.y || (a.y_stride % V == 0 && on(a.y, V * yb)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.x_dtype == OPUS_DTYPE_F32) {
    if (a.y_dtype == OPUS_DTYPE_F32) return launch_by_width<float, float>(a, vec, st);
    if (a.y_dtype == OPUS_DTYPE_F16) return launch_by_width<float, __half>(a, vec, st);
    return launch_by_width<float, __nv_bfloat16>(a, vec, st);
  }
  if (a.x_dtype == OPUS_DTYPE_F16) return launch_by_width<__half, __half>(a, vec, st);
  return launch_by_width<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
}
