// Residual norm, backward.
//
// With hh = (h - mean) / sd the normed row, a = dn o w and <.> the mean over a
// row (<a> for layer norms only):
//
//   dh = dh_in + (a - <a> - hh <a hh>) / sd
//   dx = r dh;  dz = g o dh;  dg = sum dh o z;  dw = sum dn o hh;  db = sum dn
//   dy = dz, or through the norm of y: c = dz o w_post,
//   dy = (c - <c> - yh <c yh>) / sd_y;  dw_post = sum dz o yh;  db_post = sum dz
//
// Rows (dx, dy) come from one kernel, sums over rows from another that reads
// the rows again: each thread keeps a column's sums over a run of rows in f32,
// runs meet in a third kernel, always in the same order.
#include "residual_norm.cuh"

namespace opus {
namespace {

template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(norm_threads(V, NV))
    rows_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a,
                            float2* __restrict__ means) {
  extern __shared__ float shared[];
  GroupSum sum(shared, s.group);
  const int t = threadIdx.x % s.group;
  const int64_t in_block = threadIdx.x / s.group;
  const TX* hp = static_cast<const TX*>(a.h);
  const TY* y = static_cast<const TY*>(a.y);
  const TY* dnp = static_cast<const TY*>(a.grad_n);
  const TX* dhp = static_cast<const TX*>(a.grad_h);
  TX* dx = static_cast<TX*>(a.grad_x);
  TY* dy = static_cast<TY*>(a.grad_y);
  const float inv_d = 1.0f / static_cast<float>(s.d);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * s.groups; base < s.rows;
       base += static_cast<int64_t>(gridDim.x) * s.groups) {
    const int64_t row = base + in_block;
    const bool live = row < s.rows;
    const float4 st = live ? reinterpret_cast<const float4*>(a.stats)[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    float hat[NV][V], g[NV][V];
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) hat[k][i] = g[k][i] = 0.f;
      if (!live || col >= s.d) continue;
      load_vec<TX, V>(hp + row * a.h_stride + col, hat[k]);
      if (dnp != nullptr) load_vec<TY, V>(dnp + row * a.grad_n_stride + col, g[k]);
      float w[V];
      load_param<V>(a.weight, a.weight_dtype, col, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hat[k][i] = (hat[k][i] - st.x) * st.y;
        g[k][i] *= w[i];
        m[0] += g[k][i];
        m[1] = fmaf(g[k][i], hat[k][i], m[1]);
      }
    }
    sum(m);
    m[0] = s.layer ? m[0] * inv_d : 0.f;
    m[1] *= inv_d;
    if (live && t == 0 && means != nullptr) means[row] = make_float2(m[0], m[1]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
      if (!live || col >= s.d) continue;
      float in[V];
#pragma unroll
      for (int i = 0; i < V; ++i) in[i] = 0.f;
      if (dhp != nullptr) load_vec<TX, V>(dhp + row * a.grad_h_stride + col, in);
      float out[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        g[k][i] = in[i] + st.y * (g[k][i] - m[0] - hat[k][i] * m[1]);
        out[i] = a.residual_scale * g[k][i];
      }
      store_vec<TX, V>(dx + row * s.d + col, out);
      if (y != nullptr && a.gate != nullptr) {
        float q[V];
        load_param<V>(a.gate, a.gate_dtype, row / s.seq * s.d + col, 1.f, q);
#pragma unroll
        for (int i = 0; i < V; ++i) g[k][i] *= q[i];
      }
      if (y != nullptr && !a.post) store_vec<TY, V>(dy + row * s.d + col, g[k]);
    }
    if (!a.post) continue;
    float p[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
      if (!live || col >= s.d) continue;
      float w[V];
      load_vec<TY, V>(y + row * a.y_stride + col, hat[k]);
      load_param<V>(a.post_weight, a.post_weight_dtype, col, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hat[k][i] = (hat[k][i] - st.z) * st.w;
        g[k][i] *= w[i];
        p[0] += g[k][i];
        p[1] = fmaf(g[k][i], hat[k][i], p[1]);
      }
    }
    sum(p);
    p[0] = s.layer ? p[0] * inv_d : 0.f;
    p[1] *= inv_d;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * s.group + t) * V;
      if (!live || col >= s.d) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) g[k][i] = st.w * (g[k][i] - p[0] - hat[k][i] * p[1]);
      store_vec<TY, V>(dy + row * s.d + col, g[k]);
    }
  }
}

enum Column : int { kWeight = 0, kBias, kPostWeight, kPostBias, kGate, kColumns };

constexpr int kColWarps = 8;
constexpr int kRun = 64;  // rows of a run at least

// One block: 32 * V columns, one run of rows.  parts[run][array][d].
template <typename TX, typename TY, int V>
__global__ void __launch_bounds__(kColWarps * 32)
    columns_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a,
                   const float2* __restrict__ means, int wanted, int64_t seq, int64_t run, int runs_per_seq,
                   float* __restrict__ parts) {
  __shared__ float meet[kColWarps][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * V;
  const int64_t sample = blockIdx.x / runs_per_seq;
  const int64_t first = sample * seq + (blockIdx.x % runs_per_seq) * run;
  const int64_t last = first + run < (sample + 1) * seq ? first + run : (sample + 1) * seq;
  const bool own = col < s.d;
  float acc[kColumns][V];
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[c][i] = 0.f;
  const bool deep = (wanted & (1 << kPostWeight | 1 << kPostBias | 1 << kGate)) != 0;
  if (own) {
    float w[V], pw[V], pb[V];
    load_param<V>(a.weight, a.weight_dtype, col, 1.f, w);
    load_param<V>(a.post_weight, a.post_weight_dtype, col, 1.f, pw);
    load_param<V>(a.post_bias, a.post_bias_dtype, col, 0.f, pb);
    for (int64_t row = first + warp; row < last; row += kColWarps) {
      const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
      float hat[V], dn[V];
      load_vec<TX, V>(static_cast<const TX*>(a.h) + row * a.h_stride + col, hat);
#pragma unroll
      for (int i = 0; i < V; ++i) dn[i] = 0.f;
      if (a.grad_n != nullptr) load_vec<TY, V>(static_cast<const TY*>(a.grad_n) + row * a.grad_n_stride + col, dn);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hat[i] = (hat[i] - st.x) * st.y;
        acc[kWeight][i] = fmaf(dn[i], hat[i], acc[kWeight][i]);
        acc[kBias][i] += dn[i];
      }
      if (!deep) continue;
      const float2 m = means[row];
      float dh[V], z[V], g[V];
#pragma unroll
      for (int i = 0; i < V; ++i) dh[i] = 0.f;
      if (a.grad_h != nullptr) load_vec<TX, V>(static_cast<const TX*>(a.grad_h) + row * a.grad_h_stride + col, dh);
      load_vec<TY, V>(static_cast<const TY*>(a.y) + row * a.y_stride + col, z);
      load_param<V>(a.gate, a.gate_dtype, row / s.seq * s.d + col, 1.f, g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dh[i] += st.y * (dn[i] * w[i] - m.x - hat[i] * m.y);
        if (a.post) {
          const float yh = (z[i] - st.z) * st.w;
          acc[kPostWeight][i] = fmaf(g[i] * dh[i], yh, acc[kPostWeight][i]);
          acc[kPostBias][i] = fmaf(g[i], dh[i], acc[kPostBias][i]);
          z[i] = yh * pw[i] + pb[i];
        }
        acc[kGate][i] = fmaf(dh[i], z[i], acc[kGate][i]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    if ((wanted & (1 << c)) == 0) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) meet[warp][lane * V + i] = acc[c][i];
    __syncthreads();
    if (warp != 0 || !own) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = meet[0][lane * V + i];
#pragma unroll
      for (int u = 1; u < kColWarps; ++u) v += meet[u][lane * V + i];
      parts[(static_cast<int64_t>(blockIdx.x) * kColumns + c) * s.d + col + i] = v;
    }
  }
}

struct ColumnOutputs {
  void* p[kColumns];
  int dtype[kColumns];
};

// Sums the runs of 32 columns of one array (blockIdx.y) and one sample (blockIdx.z).
__global__ void __launch_bounds__(256) columns_join_kernel(const float* __restrict__ parts, int64_t runs, int d,
                                                           const __grid_constant__ ColumnOutputs out) {
  __shared__ float meet[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane, c = blockIdx.y;
  if (out.p[c] == nullptr) return;
  const int64_t first = blockIdx.z * runs;
  float v = 0.f;
  if (col < d)
    for (int64_t r = runs * slice / 8; r < runs * (slice + 1) / 8; ++r) v += parts[((first + r) * kColumns + c) * d + col];
  meet[slice][lane] = v;
  __syncthreads();
  if (slice != 0 || col >= d) return;
#pragma unroll
  for (int u = 1; u < 8; ++u) v += meet[u][lane];
  store_any(out.p[c], out.dtype[c], blockIdx.z * static_cast<int64_t>(d) + col, v);
}

struct Runs {
  int64_t seq, run;
  int64_t samples;
  int per_seq;
};
// Runs of rows that stay inside `seq` neighbours: at least kRun rows each, and about a thousand in all.
Runs runs_of(int64_t rows, int64_t seq) {
  Runs r;
  r.seq = seq;
  r.samples = seq > 0 ? rows / seq : 0;
  int64_t run = (rows + 1023) / 1024;
  r.run = run > kRun ? run : kRun;
  r.per_seq = static_cast<int>((seq + r.run - 1) / r.run);
  return r;
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

template <typename TX, typename TY, int V>
int launch_columns(const NormShape& s, const opus_residual_norm_args& a, const float2* means, int wanted,
                   const Runs& r, float* parts, const ColumnOutputs& out, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(r.samples * r.per_seq), (s.d / V + 31) / 32);
  columns_kernel<TX, TY, V><<<grid, kColWarps * 32, 0, st>>>(s, a, means, wanted, r.seq, r.run, r.per_seq, parts);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  ColumnOutputs o = out;
  for (int c = 0; c < kColumns; ++c)
    if ((wanted & (1 << c)) == 0) o.p[c] = nullptr;
  // gates of many samples go in slices of the grid's z limit
  for (int64_t at = 0; at < r.samples; at += 65535) {
    const int64_t n = r.samples - at < 65535 ? r.samples - at : 65535;
    columns_join_kernel<<<dim3((s.d + 31) / 32, kColumns, static_cast<unsigned>(n)), 256, 0, st>>>(
        parts + at * r.per_seq * kColumns * s.d, r.per_seq, s.d, o);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    if (o.p[kGate]) o.p[kGate] = static_cast<uint8_t*>(o.p[kGate]) + n * s.d * dtype_bytes(o.dtype[kGate]);
  }
  return OPUS_OK;
}

template <typename TX, typename TY, int V, int NV>
int launch(const NormShape& s, const opus_residual_norm_args& a, int wanted, uint8_t* ws, cudaStream_t st) {
  float2* means = reinterpret_cast<float2*>(ws);
  float* parts = reinterpret_cast<float*>(ws + align256(s.rows * 8));
  const int threads = (s.group * s.groups + 31) / 32 * 32;
  int64_t blocks = (s.rows + s.groups - 1) / s.groups;
  const int64_t most = static_cast<int64_t>(sm_count()) * (2048 / threads);
  if (blocks > most) blocks = most;
  rows_kernel<TX, TY, V, NV><<<static_cast<unsigned>(blocks), threads, 4 * (threads / 32) * sizeof(float), st>>>(s, a, means);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  const ColumnOutputs out{{a.grad_weight, a.grad_bias, a.grad_post_weight, a.grad_post_bias, a.grad_gate},
                          {a.weight_dtype, a.bias_dtype, a.post_weight_dtype, a.post_bias_dtype, a.gate_dtype}};
  // sums over all rows, then the gates of several samples in runs of their own
  const bool gates = a.gate_rows > 1 && (wanted & (1 << kGate)) != 0;
  const int whole = gates ? wanted & ~(1 << kGate) : wanted;
  if (whole != 0) {
    const int rc = launch_columns<TX, TY, V>(s, a, means, whole, runs_of(s.rows, s.rows), parts, out, st);
    if (rc) return rc;
  }
  if (gates) return launch_columns<TX, TY, V>(s, a, means, 1 << kGate, runs_of(s.rows, s.seq), parts, out, st);
  return OPUS_OK;
}

template <typename TX, typename TY>
int launch_by_width(const opus_residual_norm_args& a, bool vec, int wanted, uint8_t* ws, cudaStream_t st) {
  constexpr int V = 16 / sizeof(TX);
  NormShape s;
  int nv;
  const int rc = norm_shape("residual_norm_grad", &a, vec, V, &s, &nv);
  if (rc) return rc;
  if (!vec) return nv == 4 ? launch<TX, TY, 1, 4>(s, a, wanted, ws, st) : launch<TX, TY, 1, 16>(s, a, wanted, ws, st);
  if (nv == 1) return launch<TX, TY, V, 1>(s, a, wanted, ws, st);
  if (nv == 2) return launch<TX, TY, V, 2>(s, a, wanted, ws, st);
  if constexpr (V == 4) return launch<TX, TY, V, 4>(s, a, wanted, ws, st);
  return set_error(OPUS_ERR_UNSUPPORTED, "residual_norm_grad: d = %d", a.d);
}

bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace opus

using namespace opus;

extern "C" int64_t opus_residual_norm_grad_workspace_bytes(const opus_residual_norm_args* a) {
  if (a == nullptr || a->rows <= 0 || a->d < 1) return 256;
  const Runs whole = runs_of(a->rows, a->rows);
  int64_t runs = whole.samples * whole.per_seq;
  if (a->gate != nullptr && a->gate_rows > 1 && a->rows % a->gate_rows == 0) {
    const Runs r = runs_of(a->rows, a->rows / a->gate_rows);
    if (r.samples * r.per_seq > runs) runs = r.samples * r.per_seq;
  }
  return align256(a->rows * 8) + align256(runs * kColumns * a->d * 4);
}

extern "C" int opus_residual_norm_grad(const opus_residual_norm_args* args, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  int rc = check_norm("residual_norm_grad", args);
  if (rc) return rc;
  const opus_residual_norm_args& a = *args;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  void* outs[kColumns] = {a.grad_weight, a.grad_bias, a.grad_post_weight, a.grad_post_bias, a.grad_gate};
  const void* of[kColumns] = {a.weight, a.bias, a.post_weight, a.post_bias, a.gate};
  const int types[kColumns] = {a.weight_dtype, a.bias_dtype, a.post_weight_dtype, a.post_bias_dtype, a.gate_dtype};
  int wanted = 0;
  for (int c = 0; c < kColumns; ++c) {
    if (outs[c] == nullptr) continue;
    if (of[c] == nullptr) return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a gradient of no parameter");
    if (!on(outs[c], dtype_bytes(types[c])))
      return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a pointer is not aligned to its elements");
    wanted |= 1 << c;
    if (a.rows == 0)
      OPUS_CUDA_TRY(cudaMemsetAsync(outs[c], 0, (c == kGate ? a.gate_rows : 1) * static_cast<int64_t>(a.d) * dtype_bytes(types[c]), st));
  }
  if (a.rows == 0) return OPUS_OK;
  if (!a.h || !a.stats || !a.grad_x || (!a.grad_n && !a.grad_h) || (a.y != nullptr && a.grad_y == nullptr) ||
      (a.y == nullptr && a.grad_y != nullptr) || !workspace)
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: NULL pointer");
  if (workspace_bytes < opus_residual_norm_grad_workspace_bytes(&a))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
                     (long long)opus_residual_norm_grad_workspace_bytes(&a));
  if (!on(workspace, 256)) return set_error(OPUS_ERR_INVALID, "residual_norm_grad: workspace must be 256-byte aligned");
  const int xb = dtype_bytes(a.x_dtype), yb = dtype_bytes(a.y_dtype);
  if (a.h_stride < a.d || (a.y && a.y_stride < a.d) || (a.grad_n && a.grad_n_stride < a.d) ||
      (a.grad_h && a.grad_h_stride < a.d))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: row stride < d");
  if (!on(a.h, xb) || !on(a.grad_h, xb) || !on(a.grad_x, xb) || !on(a.y, yb) || !on(a.grad_n, yb) ||
      !on(a.grad_y, yb) || !on(a.stats, 16))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a pointer is not aligned to its elements");
  const int V = 16 / xb;
  const bool vec = a.d % V == 0 && a.h_stride % V == 0 && on(a.h, 16) && on(a.grad_x, 16) && on(a.grad_y, V * yb) &&
                   (!a.y || (a.y_stride % V == 0 && on(a.y, V * yb))) &&
                   (!a.grad_n || (a.grad_n_stride % V == 0 && on(a.grad_n, V * yb))) &&
                   (!a.grad_h || (a.grad_h_stride % V == 0 && on(a.grad_h, 16)));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (a.x_dtype == OPUS_DTYPE_F32) {
    if (a.y_dtype == OPUS_DTYPE_F32) return launch_by_width<float, float>(a, vec, wanted, ws, st);
    if (a.y_dtype == OPUS_DTYPE_F16) return launch_by_width<float, __half>(a, vec, wanted, ws, st);
    return launch_by_width<float, __nv_bfloat16>(a, vec, wanted, ws, st);
  }
  if (a.x_dtype == OPUS_DTYPE_F16) return launch_by_width<__half, __half>(a, vec, wanted, ws, st);
  return launch_by_width<__nv_bfloat16, __nv_bfloat16>(a, vec, wanted, ws, st);
}
