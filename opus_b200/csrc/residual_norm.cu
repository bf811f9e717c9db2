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

// Vector loads of the parameters need their arrays on 16-byte boundaries.
bool norm_params_aligned(const opus_residual_norm_args* a) {
  const void* p[5] = {a->weight, a->bias, a->post_weight, a->post_bias, a->gate};
  for (const void* q : p)
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return false;
  return true;
}

// The launch's shape for vectors of V elements, at most `most` of them (a power of two) a thread: as few threads
// a row as that allows, and as few vectors a thread as those threads need.
int norm_shape(const char* what, const opus_residual_norm_args* a, int V, int most, NormShape* s, int* nv) {
  const int full = (a->d + V - 1) / V;
  int group = 1;
  while (group < 32 && group * most < full) group <<= 1;
  if (group * most < full) group = ((full + most - 1) / most + 31) / 32 * 32;
  // rows of less than a warp: a vector for each lane, so that its loads are neighbours
  while (group < 32 && group < full) group <<= 1;
  if (group > kNormMaxThreads) return set_error(OPUS_ERR_UNSUPPORTED, "%s: d = %d is too wide", what, a->d);
  int k = 1;
  while (k * group < full) k <<= 1;
  *nv = k;
  s->rows = a->rows;
  s->seq = a->gate != nullptr && a->gate_rows > 1 ? a->rows / a->gate_rows : a->rows;
  if (s->seq < 1) s->seq = 1;
  s->d = a->d;
  s->group = group;
  s->groups = group >= 256 ? 1 : 256 / group;
  s->layer = a->kind;
  s->eps = a->eps;
  s->blocks = 0;
  return OPUS_OK;
}

namespace {

enum Form : int { kAlone, kJoin, kFull };  // no y; y; y with a norm or a gate

template <typename TX, typename TY, int V, int NV, int F, bool Near, bool Wide>
__global__ void __launch_bounds__(norm_threads(V, Wide), Wide ? 1 : F == kFull || V < 8 ? 2 : 3)
    residual_norm_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a) {
  extern __shared__ __align__(16) float shared[];
  const int t = threadIdx.x % s.group;
  const int g = threadIdx.x / s.group;
  const RowRun run(s.rows, static_cast<int64_t>(blockIdx.x) * s.groups + g, static_cast<int64_t>(s.blocks) * s.groups);
  const Columns<V, NV> c(s, t);
  const TX* x = static_cast<const TX*>(a.x) + run.first * a.x_stride;
  const TY* y = static_cast<const TY*>(a.y) + (F != kAlone ? run.first * a.y_stride : 0);
  TX* hp = static_cast<TX*>(a.h) + run.first * s.d;
  TY* np = static_cast<TY*>(a.n) + run.first * s.d;
  RawRow<TX, V, NV> xr;
  RawRow<TY, V, NV> yr;
  xr.zero();
  yr.zero();
  if (run.first < run.last) {
    xr.load(x, c);
    if constexpr (F != kAlone) yr.load(y, c);
  }
  GroupSum<norm_sub_warp(V, NV)> sum(shared, s.group, s.groups);
  float* place = shared + group_floats(s.group, s.groups);
  Param<NV, V, Near> w(a.weight, a.weight_dtype, 1.f), b(a.bias, a.bias_dtype, 0.f);
  Param<NV, V, Near> pw(a.post_weight, a.post_weight_dtype, 1.f), pb(a.post_bias, a.post_bias_dtype, 0.f);
  Param<NV, V, Near> q(a.gate, a.gate_dtype, 1.f);
  w.fill(&place, s);
  b.fill(&place, s);
  const bool one_gate = s.seq == s.rows;
  if constexpr (F == kFull) {
    pw.fill(&place, s);
    pb.fill(&place, s);
    if (one_gate) q.fill(&place, s);
  }
  __syncthreads();
  int64_t until = 0, gate_at = 0;  // the first row of the next sample, this sample's gate
  for (int64_t row = run.first; row < run.last; ++row) {
    float h[NV][V], u[NV][V];
    xr.get(h);
    if constexpr (F != kAlone) yr.get(u);
    x += a.x_stride;
    if constexpr (F != kAlone) y += a.y_stride;
    if (row + 1 < run.last) {
      xr.load(x, c);
      if constexpr (F != kAlone) yr.load(y, c);
    }
    float2 ys = make_float2(0.f, 1.f);
    if constexpr (F == kFull) {
      float p[NV][V];
      if (a.post) {
        ys = row_stats(u, s, c, t, sum);
        float o[NV][V];
        pw.row(c, p);
        pb.row(c, o);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) u[k][j] = fmaf((u[k][j] - ys.x) * ys.y, p[k][j], o[k][j]);
      }
      if (one_gate) {
        q.row(c, p);
      } else {
        if (row >= until) {
          gate_at = row / s.seq * s.d;
          until = (row / s.seq + 1) * s.seq;
        }
        load_param_row(a.gate, a.gate_dtype, gate_at, 1.f, c, p);
      }
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) u[k][j] *= p[k][j];
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) h[k][j] = F == kAlone ? a.residual_scale * h[k][j] : fmaf(a.residual_scale, h[k][j], u[k][j]);
      Vec<TX, V> stored;
      stored.set(h[k]);
      stored.get(h[k]);  // what is normed is what is stored
      if (c.own[k] && (F != kAlone || a.h != nullptr)) *reinterpret_cast<Vec<TX, V>*>(hp + c.at[k]) = stored;
    }
    hp += s.d;
    const float2 hs = row_stats(h, s, c, t, sum);
    float o[NV][V];
    w.row(c, u);
    b.row(c, o);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) h[k][j] = fmaf((h[k][j] - hs.x) * hs.y, u[k][j], o[k][j]);
    store_row(np, c, h);
    np += s.d;
    if (t == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(hs.x, hs.y, ys.x, ys.y);
  }
}

template <typename TX, typename TY, int V, int NV, int F, bool Near, bool Wide>
int launch(NormShape s, const opus_residual_norm_args& a, cudaStream_t st) {
  constexpr auto kernel = residual_norm_kernel<TX, TY, V, NV, F, Near, Wide>;
  const int threads = s.group * s.groups;
  const int arrays = F != kFull ? 2 : s.seq == s.rows ? 5 : 4;
  const int shared = (group_floats(s.group, s.groups) + arrays * Param<NV, V, Near>::size(s.group)) * static_cast<int>(sizeof(float));
  const int rc = allow_shared<kernel>(shared);
  if (rc) return rc;
  const int64_t need = (s.rows + s.groups - 1) / s.groups;
  const int64_t most = static_cast<int64_t>(sm_count()) * resident_blocks<kernel>(threads, shared);
  s.blocks = static_cast<int>(need < most ? need : most);
  kernel<<<s.blocks, threads, shared, st>>>(s, a);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename TX, typename TY, int V, int F>
int launch_by_width(const opus_residual_norm_args& a, cudaStream_t st) {
  constexpr int kMost = 16 / V;
  constexpr int kWide = wide_vectors(V);
  NormShape s;
  int nv;
  if (a.d > kNormNarrow) {
    const int rc = norm_shape("residual_norm", &a, V, kWide, &s, &nv);
    if (rc) return rc;
    if constexpr (F == kFull) {
      if (5 * Param<kWide, V, true>::size(s.group) * static_cast<int>(sizeof(float)) > kNormSharedParams)
        return launch<TX, TY, V, kWide, F, false, true>(s, a, st);
    }
    return launch<TX, TY, V, kWide, F, true, true>(s, a, st);
  }
  const int rc = norm_shape("residual_norm", &a, V, kMost, &s, &nv);
  if (rc) return rc;
  if constexpr (V > 1) {
    if (nv == 1) return launch<TX, TY, V, 1, F, true, false>(s, a, st);
  }
  if constexpr (V < 8) {
    if (nv <= 4 / (V == 4 ? 2 : 1)) return launch<TX, TY, V, 4 / (V == 4 ? 2 : 1), F, true, false>(s, a, st);
  }
  return launch<TX, TY, V, kMost, F, true, false>(s, a, st);
}

template <typename TX, typename TY, int V>
int launch_by_form(const opus_residual_norm_args& a, cudaStream_t st) {
  if (a.post || a.gate != nullptr) return launch_by_width<TX, TY, V, kFull>(a, st);
  if (a.y != nullptr) return launch_by_width<TX, TY, V, kJoin>(a, st);
  return launch_by_width<TX, TY, V, kAlone>(a, st);
}

template <typename TX, typename TY>
int launch_by_alignment(const opus_residual_norm_args& a, bool vec, cudaStream_t st) {
  return vec ? launch_by_form<TX, TY, 16 / sizeof(TX)>(a, st) : launch_by_form<TX, TY, 1>(a, st);
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
  const bool vec = norm_params_aligned(&a) && a.d % V == 0 && a.x_stride % V == 0 && on(a.x, 16) && on(a.h, 16) && on(a.n, V * yb) &&
                   (!a.y || (a.y_stride % V == 0 && on(a.y, V * yb)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.x_dtype == OPUS_DTYPE_F32) {
    if (a.y_dtype == OPUS_DTYPE_F32) return launch_by_alignment<float, float>(a, vec, st);
    if (a.y_dtype == OPUS_DTYPE_F16) return launch_by_alignment<float, __half>(a, vec, st);
    return launch_by_alignment<float, __nv_bfloat16>(a, vec, st);
  }
  if (a.x_dtype == OPUS_DTYPE_F16) return launch_by_alignment<__half, __half>(a, vec, st);
  return launch_by_alignment<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
}
