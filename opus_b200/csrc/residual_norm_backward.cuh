// Residual norm, backward: kernels and their launch, for one pair of types (included by residual_norm_<types>.cu).
//
// With hh = (h - mean) / sd the normed row, a = dn o w and <.> the mean over a
// row (<a> for layer norms only):
//
//   dh = dh_in + (a - <a> - hh <a hh>) / sd
//   dx = r dh;  dz = g o dh;  dg = sum dh o z;  dw = sum dn o hh;  db = sum dn
//   dy = dz, or through the norm of y: c = dz o w_post,
//   dy = (c - <c> - yh <c yh>) / sd_y;  dw_post = sum dz o yh;  db_post = sum dz
//
// Narrow rows (norm_narrow: d up to 4096 or 2048): one kernel reads each row once, writes dx and dy, and keeps a
// column's sums over its run of rows in registers (16 columns a thread, five
// sums each); a second kernel joins the runs.  Wider rows would need more
// than 256 threads and leave them too few registers for that: one kernel for
// dx and dy, another that reads the rows again for the sums, and the same
// join.  Every sum has a fixed order.
//
// Bound: HBM bandwidth (h, dn, dh_in and y read once, dx and dy written once).
// 65536 x 2048 bf16: RMS joints 210 us, 6.4 TB/s; layer norms with biases 267 us,
// 5.0 TB/s (161 registers: one block an SM); both norms and a gate 369 us, 4.4
// TB/s (241 registers: eight warps an SM, a third of the issue slots).  8 elements
// a thread would leave room for twice the warps and took 535 us.  32768 x 2048 f32:
// 213 us, 6.3 TB/s.  Wide rows are read twice: 8192 x 8192 f32 356 us, 3.8 TB/s.
#pragma once

#include "residual_norm.cuh"

namespace opus {
namespace {

// The worker (group of threads) whose run of rows holds `row`: RowRun's split, inverted.
__device__ __forceinline__ int64_t worker_of(int64_t row, int64_t rows, int64_t n) {
  const int64_t each = rows / n, more = rows % n, cut = more * (each + 1);
  return row < cut ? row / (each + 1) : more + (row - cut) / each;
}

// parts[block][array][d]: sums over the block's rows.  gates[worker + sample][d]: sums over the worker's rows of
// one sample, where each sample has a gate (a step to the next worker or sample is a step to the next slot).
// Full: with a norm of y or a gate.  Bias: sums for bias and post_bias too.
template <typename TX, typename TY, int V, int NV, bool Full, bool Bias>
__global__ void __launch_bounds__(norm_threads(V, false))
    grad_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a, int wanted,
                float* __restrict__ parts, float* __restrict__ gates) {
  extern __shared__ __align__(16) float shared[];
  constexpr bool kPairs = V == 8;
  const int t = threadIdx.x % s.group;
  const int g = threadIdx.x / s.group;
  const int64_t worker = static_cast<int64_t>(blockIdx.x) * s.groups + g;
  const RowRun run(s.rows, worker, static_cast<int64_t>(s.blocks) * s.groups);
  const Columns<V, NV> c(s, t);
  const TX* hp = static_cast<const TX*>(a.h) + run.first * a.h_stride;
  const TX* dhp = static_cast<const TX*>(a.grad_h) + run.first * a.grad_h_stride;
  const TY* dnp = static_cast<const TY*>(a.grad_n) + run.first * a.grad_n_stride;
  const TY* yp = static_cast<const TY*>(a.y) + run.first * a.y_stride;
  TX* dx = static_cast<TX*>(a.grad_x) + run.first * s.d;
  TY* dy = static_cast<TY*>(a.grad_y) + run.first * s.d;
  const float4* stats = reinterpret_cast<const float4*>(a.stats) + run.first;
  RawRow<TX, V, NV> hr, dhr;
  RawRow<TY, V, NV> dnr, yr;
  float4 ahead = make_float4(0.f, 0.f, 0.f, 0.f);
  hr.zero(), dhr.zero(), dnr.zero(), yr.zero();
  const auto fetch = [&]() {
    hr.load(hp, c);
    if (a.grad_n != nullptr) dnr.load(dnp, c);
    if (a.grad_h != nullptr) dhr.load(dhp, c);
    if constexpr (Full) yr.load(yp, c);
    ahead = *stats;
    hp += a.h_stride, dhp += a.grad_h_stride, dnp += a.grad_n_stride, yp += a.y_stride, ++stats;
  };
  if (run.first < run.last) fetch();
  GroupSum<norm_sub_warp(V, NV)> sum(shared, s.group, s.groups);
  float* meet = shared + group_floats(s.group, s.groups);
  float* place = meet + (s.groups > 1 ? blockDim.x * V * NV : 0);
  const bool one_gate = s.seq == s.rows;
  Param<NV, V, true> w(a.weight, a.weight_dtype, 1.f), q(a.gate, a.gate_dtype, 1.f);
  Param<NV, V, true> pw(a.post_weight, a.post_weight_dtype, 1.f), pb(a.post_bias, a.post_bias_dtype, 0.f);
  w.fill(&place, s);
  if constexpr (Full) {
    pw.fill(&place, s);
    if constexpr (Bias) pb.fill(&place, s);
    if (one_gate) q.fill(&place, s);
  }
  __syncthreads();
  const float inv_d = 1.0f / static_cast<float>(s.d);
  float acc_w[NV][V], acc_b[Bias ? NV : 1][V], acc_pw[Full ? NV : 1][V], acc_pb[Full && Bias ? NV : 1][V], acc_g[Full ? NV : 1][V];
  const auto clear = [](auto& acc) {
    for (auto& k : acc)
      for (float& v : k) v = 0.f;
  };
  clear(acc_w), clear(acc_b), clear(acc_pw), clear(acc_pb), clear(acc_g);
  int64_t sample = -1, until = -1;  // of the gate whose sums are held; the first row of the next sample
  const auto flush_gate = [&]() {
    if constexpr (Full) {
      if (sample < 0 || (wanted & (1 << kGate)) == 0) return;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (c.own[k]) store_vec<float, V>(gates + (worker + sample) * s.d + c.at[k], acc_g[k]);
      }
      clear(acc_g);
    }
  };
  for (int64_t row = run.first; row < run.last; ++row) {
    float hat[NV][V], u[NV][V], r[NV][V], y[NV][V], f[NV][V];
    hr.get(hat);
    dnr.get(u);
    dhr.get(r);
    if constexpr (Full) yr.get(y);
    const float4 st = ahead;
    if (row + 1 < run.last) fetch();
    float m[2], m0[2] = {0.f, 0.f}, m1[2] = {0.f, 0.f};
    w.row(c, f);
    normalize<kPairs>(hat, st.x, st.y);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      vmac<kPairs>(acc_w[k], u[k], hat[k]);
      if constexpr (Bias) vadd<kPairs>(acc_b[k], u[k]);
      vmul<kPairs>(u[k], f[k]);
      if (s.layer) vsum<kPairs>(m0, u[k]);
      vdot<kPairs>(m1, u[k], hat[k]);
    }
    m[0] = m0[0] + m0[1];
    m[1] = m1[0] + m1[1];
    sum(m, t);
    // dh in u
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      vmul<kPairs>(hat[k], -m[1] * inv_d);
      vadd<kPairs>(u[k], hat[k]);
      if (s.layer) vadd<kPairs>(u[k], -m[0] * inv_d);
      vfma<kPairs>(u[k], st.y, r[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) r[k][j] = u[k][j];
      vmul<kPairs>(r[k], a.residual_scale);
    }
    store_row(dx, c, r);
    dx += s.d;
    if constexpr (Full) {
      if (one_gate) {
        q.row(c, r);
      } else {
        if (row >= until) {
          flush_gate();
          sample = row / s.seq;
          until = (sample + 1) * s.seq;
        }
        load_param_row(a.gate, a.gate_dtype, sample * s.d, 1.f, c, r);
      }
      if (!a.post) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          vmac<kPairs>(acc_g[k], u[k], y[k]);
          vmul<kPairs>(u[k], r[k]);
        }
      } else {
        pw.row(c, f);
        if constexpr (Bias) pb.row(c, hat);
        normalize<kPairs>(y, st.z, st.w);
        float p[2], p0[2] = {0.f, 0.f}, p1[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float z[V];
#pragma unroll
          for (int j = 0; j < V; ++j) z[j] = y[k][j];
          if constexpr (Bias) vfma<kPairs>(z, f[k], hat[k]);
          else vmul<kPairs>(z, f[k]);
          vmac<kPairs>(acc_g[k], u[k], z);
          vmul<kPairs>(u[k], r[k]);  // dz
          vmac<kPairs>(acc_pw[k], u[k], y[k]);
          if constexpr (Bias) vadd<kPairs>(acc_pb[k], u[k]);
          vmul<kPairs>(u[k], f[k]);
          if (s.layer) vsum<kPairs>(p0, u[k]);
          vdot<kPairs>(p1, u[k], y[k]);
        }
        p[0] = p0[0] + p0[1];
        p[1] = p1[0] + p1[1];
        sum(p, t);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          vmul<kPairs>(y[k], -p[1] * inv_d);
          vadd<kPairs>(u[k], y[k]);
          if (s.layer) vadd<kPairs>(u[k], -p[0] * inv_d);
          vmul<kPairs>(u[k], st.w);
        }
      }
    }
    if (a.grad_y != nullptr) store_row(dy, c, u);
    dy += s.d;
  }
  if (!one_gate) flush_gate();
  // the block's groups together, in order
  const auto finish = [&](auto& acc, int which) {
    if ((wanted & (1 << which)) == 0) return;
    if (s.groups > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) meet[(k * V + j) * blockDim.x + threadIdx.x] = acc[k][j];
      __syncthreads();
      if (g == 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j)
            for (int o = 1; o < s.groups; ++o) acc[k][j] += meet[(k * V + j) * blockDim.x + o * s.group + t];
      }
    }
    if (g != 0) return;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c.own[k]) store_vec<float, V>(parts + (static_cast<int64_t>(blockIdx.x) * kColumns + which) * s.d + c.at[k], acc[k]);
    }
  };
  finish(acc_w, kWeight);
  if constexpr (Bias) finish(acc_b, kBias);
  if constexpr (Full) {
    finish(acc_pw, kPostWeight);
    if constexpr (Bias) finish(acc_pb, kPostBias);
    if (one_gate) finish(acc_g, kGate);
  }
}

// ---- wider rows
template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(norm_threads(V, true))
    rows_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a,
                float2* __restrict__ means) {
  extern __shared__ __align__(16) float shared[];
  const int t = threadIdx.x % s.group;
  const int g = threadIdx.x / s.group;
  const RowRun run(s.rows, static_cast<int64_t>(blockIdx.x) * s.groups + g, static_cast<int64_t>(s.blocks) * s.groups);
  const Columns<V, NV> c(s, t);
  const float inv_d = 1.0f / static_cast<float>(s.d);
  GroupSum<false> sum(shared, s.group, s.groups);
  for (int64_t row = run.first; row < run.last; ++row) {
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    RawRow<TX, V, NV> hr, in;
    RawRow<TY, V, NV> r2;  // dn, then y
    hr.zero(), in.zero(), r2.zero();
    hr.load(static_cast<const TX*>(a.h) + row * a.h_stride, c);
    if (a.grad_n != nullptr) r2.load(static_cast<const TY*>(a.grad_n) + row * a.grad_n_stride, c);
    if (a.grad_h != nullptr) in.load(static_cast<const TX*>(a.grad_h) + row * a.grad_h_stride, c);
    float v[NV][V];
    float m[2] = {0.f, 0.f};
    load_param_row(a.weight, a.weight_dtype, 0, 1.f, c, v);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float hat[V], dn[V];
      hr.v[k].get(hat);
      r2.v[k].get(dn);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[k][j] *= dn[j];
        m[0] += v[k][j];
        m[1] = fmaf(v[k][j], (hat[j] - st.x) * st.y, m[1]);
      }
    }
    sum(m, t);
    m[0] = s.layer ? m[0] * inv_d : 0.f;
    m[1] *= inv_d;
    if (t == 0) means[row] = make_float2(m[0], m[1]);
    if (a.post) r2.load(static_cast<const TY*>(a.y) + row * a.y_stride, c);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float hat[V], r[V];
      hr.v[k].get(hat);
      in.v[k].get(r);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[k][j] = r[j] + st.y * (v[k][j] - m[0] - (hat[j] - st.x) * st.y * m[1]);
        r[j] = a.residual_scale * v[k][j];
      }
      if (c.own[k]) store_vec<TX, V>(static_cast<TX*>(a.grad_x) + row * s.d + c.at[k], r);
    }
    if (a.gate != nullptr) {
      float q[NV][V];
      load_param_row(a.gate, a.gate_dtype, s.seq != s.rows ? row / s.seq * s.d : 0, 1.f, c, q);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] *= q[k][j];
    }
    if (a.post) {
      float p[2] = {0.f, 0.f}, u[NV][V];
      load_param_row(a.post_weight, a.post_weight_dtype, 0, 1.f, c, u);  // zeros beyond the row
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float y[V];
        r2.v[k].get(y);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[k][j] *= u[k][j];
          p[0] += v[k][j];
          p[1] = fmaf(v[k][j], (y[j] - st.z) * st.w, p[1]);
        }
      }
      sum(p, t);
      p[0] = s.layer ? p[0] * inv_d : 0.f;
      p[1] *= inv_d;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float y[V];
        r2.v[k].get(y);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = st.w * (v[k][j] - p[0] - (y[j] - st.z) * st.w * p[1]);
      }
    }
    if (a.grad_y != nullptr) store_row(static_cast<TY*>(a.grad_y) + row * s.d, c, v);
  }
}

constexpr int kColWarps = 8;

template <int V>
__device__ __forceinline__ void column_param(const void* p, int dtype, int64_t at, float other, float (&r)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = other;
  if (p != nullptr) load_param_vec<V>(p, dtype, at, r);
}

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
    column_param<V>(a.weight, a.weight_dtype, col, 1.f, w);
    column_param<V>(a.post_weight, a.post_weight_dtype, col, 1.f, pw);
    column_param<V>(a.post_bias, a.post_bias_dtype, col, 0.f, pb);
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
      column_param<V>(a.gate, a.gate_dtype, (s.seq == s.rows ? 0 : row / s.seq) * s.d + col, 1.f, g);
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

constexpr int kSlices = 32;

// Sums v[first + r * stride + col] over r in [0, count) for 32 columns by the block's 32 slices; warp 0 has the result.
__device__ __forceinline__ float join_parts(const float* v, int64_t count, int64_t stride, bool own) {
  __shared__ float meet[kSlices][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  float sum = 0.f;
  if (own) {
#pragma unroll 4
    for (int64_t r = slice; r < count; r += kSlices) sum += v[r * stride];
  }
  meet[slice][lane] = sum;
  __syncthreads();
  // warp w turns slice sums of column w + ... into one: 32 slices of a column lie in one warp after the transpose
  float x = meet[lane][slice];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;  // of column `slice`, in every lane
}

// blockIdx.y < kColumns: an array of parts[run][array][d] (its sums over all runs).  Behind them the gates of samples
// first + blockIdx.y - kColumns, from gates[worker + sample][d] of `workers` groups of threads.
__global__ void __launch_bounds__(kSlices * 32) columns_join_kernel(const float* __restrict__ parts, int64_t runs, int d,
                                                                    const __grid_constant__ ColumnOutputs out,
                                                                    const float* __restrict__ gates, int64_t rows,
                                                                    int64_t seq, int64_t workers, int64_t first, void* gate) {
  wait_for_predecessors();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), at = blockIdx.x * 32 + (threadIdx.x >> 5);
  const bool writes = (threadIdx.x & 31) == 0 && at < d;
  if (blockIdx.y < kColumns) {
    const int c = blockIdx.y;
    if (out.p[c] == nullptr) return;
    const float v = join_parts(parts + static_cast<int64_t>(c) * d + col, runs, static_cast<int64_t>(kColumns) * d, col < d);
    if (writes) store_any(out.p[c], out.dtype[c], at, v);
    return;
  }
  const int64_t sample = first + blockIdx.y - kColumns;
  const int64_t a = worker_of(sample * seq, rows, workers), b = worker_of((sample + 1) * seq - 1, rows, workers);
  const float v = join_parts(gates + (a + sample) * d + col, b - a + 1, d, col < d);
  if (writes) store_any(gate, out.dtype[kGate], sample * d + at, v);
}

// The gates of wide rows: runs per_seq of each sample, array kGate of parts[run][array][d].
__global__ void __launch_bounds__(kSlices * 32) gate_runs_join_kernel(const float* __restrict__ parts, int64_t per_seq,
                                                                      int64_t first, int d, void* out, int dtype) {
  const int64_t sample = first + blockIdx.y;
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const float v = join_parts(parts + (sample * per_seq * kColumns + kGate) * d + col, per_seq,
                             static_cast<int64_t>(kColumns) * d, col < d);
  const int at = blockIdx.x * 32 + (threadIdx.x >> 5);
  if ((threadIdx.x & 31) == 0 && at < d) store_any(out, dtype, sample * d + at, v);
}

constexpr int64_t kMaxSamples = 65535 - kColumns;  // of one launch: the grid's y limit

// Joins the arrays in `wanted`, and the gates of `samples` samples into gate.
int launch_columns_join(const float* parts, int64_t runs, const NormShape& s, int wanted, ColumnOutputs out,
                        const float* gates, int64_t samples, void* gate, cudaStream_t st) {
  for (int c = 0; c < kColumns; ++c)
    if ((wanted & (1 << c)) == 0) out.p[c] = nullptr;
  const int64_t workers = static_cast<int64_t>(s.blocks) * s.groups;
  int64_t at = 0;
  do {
    const int64_t n = samples - at < kMaxSamples ? samples - at : kMaxSamples;
    const dim3 grid((s.d + 31) / 32, static_cast<unsigned>(kColumns + n));
    OPUS_CUDA_TRY(launch_early(columns_join_kernel, grid, kSlices * 32, 0, st, parts, runs, s.d, out, gates, s.rows, s.seq,
                               workers, at, gate));
    note_launch();
    for (int c = 0; c < kColumns; ++c) out.p[c] = nullptr;  // joined
    at += kMaxSamples;
  } while (at < samples);
  return OPUS_OK;
}

template <typename TX, typename TY, int V, int NV, bool Full, bool Bias>
int launch_one_pass(NormShape s, const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws,
                    cudaStream_t st) {
  constexpr auto kernel = grad_kernel<TX, TY, V, NV, Full, Bias>;
  const int threads = s.group * s.groups;
  const int arrays = !Full ? 1 : (Bias ? 3 : 2) + (s.seq == s.rows ? 1 : 0);
  const int shared = (group_floats(s.group, s.groups) + (s.groups > 1 ? threads * V * NV : 0) +
                      arrays * Param<NV, V, true>::size(s.group)) * static_cast<int>(sizeof(float));
  const int ready = allow_shared<kernel>(shared);
  if (ready) return ready;
  int per_sm = resident_blocks<kernel>(threads, shared);
  per_sm = per_sm < kGradBlocksPerSm ? per_sm : kGradBlocksPerSm;
  const int64_t need = (s.rows + s.groups - 1) / s.groups, most = static_cast<int64_t>(sm_count()) * per_sm;
  s.blocks = static_cast<int>(need < most ? need : most);
  float* parts = reinterpret_cast<float*>(ws);
  float* gates = parts + static_cast<int64_t>(s.blocks) * kColumns * s.d;
  kernel<<<s.blocks, threads, shared, st>>>(s, a, wanted, parts, gates);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  const bool per_sample = s.seq != s.rows && (wanted & (1 << kGate)) != 0;
  const int whole = per_sample ? wanted & ~(1 << kGate) : wanted;
  if (wanted == 0) return OPUS_OK;
  return launch_columns_join(parts, s.blocks, s, whole, out, gates, per_sample ? a.gate_rows : 0, a.grad_gate, st);
}

template <typename TX, typename TY, int V>
int launch_columns(const NormShape& s, const opus_residual_norm_args& a, const float2* means, int wanted,
                   const Runs& r, float* parts, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(r.samples * r.per_seq), (s.d / V + 31) / 32);
  columns_kernel<TX, TY, V><<<grid, kColWarps * 32, 0, st>>>(s, a, means, wanted, r.seq, r.run, r.per_seq, parts);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename TX, typename TY, int V, int NV>
int backward_wide(const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws, cudaStream_t st) {
  NormShape s;
  int nv;
  const int shaped = norm_shape("residual_norm_grad", &a, V, NV, &s, &nv);
  if (shaped) return shaped;
  float2* means = reinterpret_cast<float2*>(ws);
  float* parts = reinterpret_cast<float*>(ws + align256(s.rows * 8));
  constexpr auto kernel = rows_kernel<TX, TY, V, NV>;
  const int threads = s.group * s.groups;
  const int shared = group_floats(s.group, s.groups) * static_cast<int>(sizeof(float));
  const int64_t need = (s.rows + s.groups - 1) / s.groups;
  const int64_t most = static_cast<int64_t>(sm_count()) * resident_blocks<kernel>(threads, shared);
  s.blocks = static_cast<int>(need < most ? need : most);
  kernel<<<s.blocks, threads, shared, st>>>(s, a, means);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  // sums over all rows, then the gates of several samples in runs of their own
  const bool per_sample = s.seq != s.rows && (wanted & (1 << kGate)) != 0;
  const int whole = per_sample ? wanted & ~(1 << kGate) : wanted;
  int rc = OPUS_OK;
  if (whole != 0) {
    const Runs r = runs_of(s.rows, s.rows);
    rc = launch_columns<TX, TY, V>(s, a, means, whole, r, parts, st);
    if (rc == OPUS_OK) rc = launch_columns_join(parts, r.per_seq, s, whole, out, nullptr, 0, nullptr, st);
  }
  if (rc || !per_sample) return rc;
  const Runs r = runs_of(s.rows, s.seq);
  rc = launch_columns<TX, TY, V>(s, a, means, 1 << kGate, r, parts, st);
  for (int64_t at = 0; rc == OPUS_OK && at < r.samples; at += kMaxSamples) {
    const int64_t n = r.samples - at < kMaxSamples ? r.samples - at : kMaxSamples;
    gate_runs_join_kernel<<<dim3((s.d + 31) / 32, static_cast<unsigned>(n)), kSlices * 32, 0, st>>>(
        parts, r.per_seq, at, s.d, a.grad_gate, a.gate_dtype);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
  }
  return rc;
}

template <typename TX, typename TY, int V, bool Full, bool Bias>
int backward_by_width(const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws, cudaStream_t st) {
  // 16 elements a thread, 8 where the sums of 16 f32 columns would not leave registers enough (with biases) and 8
  // reach the row's end
  constexpr int kMost = narrow_vectors(V, Full), kFewer = fewer_vectors(V, Full);
  constexpr bool kLean = V == 4 && Full && Bias;
  NormShape s;
  int nv;
  const bool lean = kLean && a.d <= norm_narrow(V, Full) / 2;
  const int rc = norm_shape("residual_norm_grad", &a, V, lean ? kFewer : kMost, &s, &nv);
  if (rc) return rc;
  if constexpr (V > 1) {
    if (nv == 1) return launch_one_pass<TX, TY, V, 1, Full, Bias>(s, a, wanted, out, ws, st);
  }
  if constexpr (V < 8) {
    if (nv <= kFewer) return launch_one_pass<TX, TY, V, kFewer, Full, Bias>(s, a, wanted, out, ws, st);
  }
  return launch_one_pass<TX, TY, V, kMost, Full, Bias>(s, a, wanted, out, ws, st);
}

template <typename TX, typename TY, int V>
int backward_by_form(const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws, cudaStream_t st) {
  const bool full = a.post || a.gate != nullptr;
  if (a.d > norm_narrow(V, full)) {
    return a.d <= kNormMiddle ? backward_wide<TX, TY, V, middle_vectors(V)>(a, wanted, out, ws, st)
                              : backward_wide<TX, TY, V, 2 * middle_vectors(V)>(a, wanted, out, ws, st);
  }
  const bool bias = a.post_bias != nullptr || (wanted & (1 << kBias)) != 0;
  if (full)
    return bias ? backward_by_width<TX, TY, V, true, true>(a, wanted, out, ws, st)
                : backward_by_width<TX, TY, V, true, false>(a, wanted, out, ws, st);
  return bias ? backward_by_width<TX, TY, V, false, true>(a, wanted, out, ws, st)
              : backward_by_width<TX, TY, V, false, false>(a, wanted, out, ws, st);
}

template <typename TX, typename TY>
int backward_by_alignment(const opus_residual_norm_args& a, bool vec, int wanted, const ColumnOutputs& out, uint8_t* ws,
                        cudaStream_t st) {
  return vec ? backward_by_form<TX, TY, 16 / sizeof(TX)>(a, wanted, out, ws, st)
             : backward_by_form<TX, TY, 1>(a, wanted, out, ws, st);
}

}  // namespace
}  // namespace opus
