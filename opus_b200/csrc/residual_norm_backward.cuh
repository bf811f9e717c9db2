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
// One kernel reads each row once, writes dx and dy, and keeps a column's sums
// over its run of rows in registers (16 columns a thread, up to five sums each); a
// second kernel joins the runs.  Blocks of 512 threads would have too few
// registers for that (all but one form have 256, that one 384): rows wider than
// 256 threads hold (4096 elements, or 2048) are split among the blocks of a
// cluster, which exchange the row's sums through each other's shared memory.
// Every sum has a fixed order.
//
// Bound: HBM bandwidth (h, dn, dh_in and y read once, dx and dy written once).
// 65536 x 2048 bf16: RMS joints 210 us, 6.4 TB/s; layer norms with biases 227 us,
// 5.9 TB/s; both norms and a gate 299 us, 5.4
// TB/s (214 registers: eight warps an SM), 368 with a third sum a column for the
// gate and five parameter arrays read for every row.  8 elements a thread would
// leave room for twice the warps and took 535 us where 16 took 374.  32768 x 2048
// f32: 213 us, 6.3 TB/s; both norms and a gate 252 us, 6.4 TB/s.  Wide rows, 8192
// x 8192: bf16 RMS 115 us (5.8 TB/s), both norms and a gate 230 (3.5); f32 219 us
// (6.1 TB/s).  A kernel for dx and dy and
// a second read of the rows for the sums took 256, 445 and 356.
#pragma once

#include "residual_norm.cuh"

namespace opus {
namespace {

// The worker (group of threads) whose run of rows holds `row`: RowRun's split, inverted.
__device__ __forceinline__ int64_t worker_of(int64_t row, int64_t rows, int64_t n) {
  const int64_t each = rows / n, more = rows % n, cut = more * (each + 1);
  return row < cut ? row / (each + 1) : more + (row - cut) / each;
}

enum GradForm : int { kGradJoin, kGradFull, kGradSamples };  // y as it is; with a norm or one gate; a gate a sample

// Blocks that a multiprocessor's registers have to hold: two where the sums of a thread's columns leave room for them
// (16384 x 4096 bf16 RMS 111 us, 138 with the registers of one; 500000 x 128 with layer norms 136 and 185), three for
// 4 elements a thread, otherwise one, which may then use all that it needs (8192 x 8192 f32 with both layer norms
// 593 us, 674 where the compiler chose).
constexpr int grad_blocks(int V, int NV, int form, bool bias) {
  const bool full = form != kGradJoin;
  const int elements = V * NV;
  if (elements <= 4) return full ? 2 : 3;
  if (elements <= 8) return !full || (V == 8 && !bias) ? 2 : 1;
  return V == 8 && !full && !bias ? 2 : 1;
}

// Threads of a block: 384 where their registers (168 a thread) fill a multiprocessor that a block of 256 would leave a
// third of (24576 x 1600 bf16 layer norms 86 us, 98 with 256; 65536 x 2048 227 and 264).
constexpr int kGradLargeThreads = 384;
static_assert(kGradLargeThreads <= kNormMostThreads, "groups of a block");
constexpr int grad_threads(int V, int NV, int form, bool bias, bool wide) {
  return V == 8 && NV == 2 && form == kGradJoin && bias && !wide ? kGradLargeThreads : kNormThreads;
}

// parts[block or cluster][array][d]: sums over its rows.  gates[worker + sample][d]: sums over the worker's rows of
// one sample, where each sample has a gate (a step to the next worker or sample is a step to the next slot).
// Bias: sums for bias and post_bias too.
// Wide: the blocks of a cluster share a row, each holding a range of its columns.
template <typename TX, typename TY, int V, int NV, int Form, bool Bias, bool Wide>
__global__ void __launch_bounds__(grad_threads(V, NV, Form, Bias, Wide), grad_blocks(V, NV, Form, Bias))
    grad_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a, int wanted,
                float* __restrict__ parts, float* __restrict__ gates) {
  extern __shared__ __align__(16) float shared[];
  constexpr bool kPairs = V == 8;
  constexpr bool Full = Form != kGradJoin, Samples = Form == kGradSamples;
  const int t = threadIdx.x % s.group;
  const int g = threadIdx.x / s.group;
  const int rank = Wide ? static_cast<int>(cluster_ctarank()) : 0;
  const int base = Wide ? rank * s.group * NV * V : 0;
  const int64_t unit = Wide ? blockIdx.x / s.ranks : blockIdx.x;
  const int64_t worker = unit * s.groups + g;
  const RowRun run(s.rows, worker, static_cast<int64_t>(s.blocks) * s.groups);
  const Columns<V, NV> c(s, t, base);
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
  GroupSum<norm_sub_warp(V, NV), Wide> sum(shared, s);
  float* meet = shared + group_floats(s.group, s.groups, Wide ? s.ranks : 1);
  float* place = meet + (s.groups > 1 ? blockDim.x * V * NV : 0);
  Param<NV, V> w(a.weight, a.weight_dtype, 1.f, base);
  Param<NV, V> pw(a.post_weight, a.post_weight_dtype, 1.f, base), pb(a.post_bias, a.post_bias_dtype, 0.f, base);
  w.fill(&place, s);
  if constexpr (Full) pw.fill(&place, s, Samples ? nullptr : a.gate, a.gate_dtype);  // g o w_post for one gate
  if constexpr (Samples && Bias) pb.fill(&place, s);
  __syncthreads();
  const float inv_d = 1.0f / static_cast<float>(s.d);
  float acc_w[NV][V], acc_b[Bias ? NV : 1][V], acc_pw[Full ? NV : 1][V], acc_pb[Full && Bias ? NV : 1][V], acc_g[Samples ? NV : 1][V];
  const auto clear = [](auto& acc) {
    for (auto& k : acc)
      for (float& v : k) v = 0.f;
  };
  clear(acc_w), clear(acc_b), clear(acc_pw), clear(acc_pb), clear(acc_g);
  int64_t sample = -1, until = -1;  // of the gate whose sums are held; the first row of the next sample
  const auto flush_gate = [&]() {
    if constexpr (Samples) {
      if (sample < 0 || (wanted & (1 << kGate)) == 0) return;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (c.own[k]) store_vec<float, V>(gates + (worker + sample) * s.d + c.at[k], acc_g[k]);
      }
      clear(acc_g);
    }
  };
  // u = (u - <u> - yh <u yh>) / sd from the sums p; yh is overwritten
  const auto through_norm = [&](float (&u)[NV][V], float (&yh)[NV][V], const float (&p)[2], float rstd) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      vmul<kPairs>(yh[k], -p[1] * inv_d);
      vadd<kPairs>(u[k], yh[k]);
      if (s.layer) vadd<kPairs>(u[k], -p[0] * inv_d);
      vmul<kPairs>(u[k], rstd);
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
    if constexpr (Form == kGradFull) {
      // One gate: dw_post = g o A, dg = w_post o A + b_post o B and db_post = g o B with A = sum dh o yh (y itself
      // without its norm) and B = sum dh, so that two sums are held, not three.
      pw.row(c, f);
      if (a.post) normalize<kPairs>(y, st.z, st.w);
      float p[2], p0[2] = {0.f, 0.f}, p1[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        vmac<kPairs>(acc_pw[k], u[k], y[k]);
        if constexpr (Bias) vadd<kPairs>(acc_pb[k], u[k]);
        vmul<kPairs>(u[k], f[k]);
        if (s.layer) vsum<kPairs>(p0, u[k]);
        vdot<kPairs>(p1, u[k], y[k]);
      }
      if (a.post) {
        p[0] = p0[0] + p0[1];
        p[1] = p1[0] + p1[1];
        sum(p, t);
        through_norm(u, y, p, st.w);
      }
    }
    if constexpr (Samples) {
      if (row >= until) {
        flush_gate();
        sample = row / s.seq;
        until = (sample + 1) * s.seq;
      }
      load_param_row(a.gate, a.gate_dtype, sample * s.d, 1.f, c, r);
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
        through_norm(u, y, p, st.w);
      }
    }
    if (a.grad_y != nullptr) store_row(dy, c, u);
    dy += s.d;
  }
  if constexpr (Samples) flush_gate();
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
      if (c.own[k]) store_vec<float, V>(parts + (unit * kColumns + which) * s.d + c.at[k], acc[k]);
    }
  };
  finish(acc_w, kWeight);
  if constexpr (Bias) finish(acc_b, kBias);
  if constexpr (Form == kGradFull) {
    float g_row[NV][V], part[NV][V];
    load_param_row(a.gate, a.gate_dtype, 0, 1.f, c, g_row);
    if ((wanted & (1 << kGate)) != 0) {
      float w_row[NV][V];
      load_param_row(a.post_weight, a.post_weight_dtype, 0, 1.f, c, w_row);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) part[k][j] = w_row[k][j] * acc_pw[k][j];
      if constexpr (Bias) {
        load_param_row(a.post_bias, a.post_bias_dtype, 0, 0.f, c, w_row);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) part[k][j] = fmaf(w_row[k][j], acc_pb[k][j], part[k][j]);
      }
      finish(part, kGate);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      vmul<kPairs>(acc_pw[k], g_row[k]);
      if constexpr (Bias) vmul<kPairs>(acc_pb[k], g_row[k]);
    }
  }
  if constexpr (Full) {
    finish(acc_pw, kPostWeight);
    if constexpr (Bias) finish(acc_pb, kPostBias);
  }
  sum.leave();
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

template <typename TX, typename TY, int V, int NV, int Form, bool Bias, bool Wide>
int launch_backward(NormShape s, const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws,
                    cudaStream_t st) {
  constexpr auto kernel = grad_kernel<TX, TY, V, NV, Form, Bias, Wide>;
  const int arrays = Form == kGradJoin ? 1 : Form == kGradSamples && Bias ? 3 : 2;
  const int shared = group_floats(s.group, s.groups, s.ranks) + (s.groups > 1 ? s.group * s.groups * V * NV : 0) +
                     arrays * Param<NV, V>::size(s.group);
  NormLaunch launch;
  const int rc = launch.plan<kernel>(&s, shared, kGradBlocksPerSm, st);
  if (rc) return rc;
  float* parts = reinterpret_cast<float*>(ws);
  float* gates = parts + static_cast<int64_t>(s.blocks) * kColumns * s.d;
  OPUS_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, kernel, s, a, wanted, parts, gates));
  note_launch();
  const bool per_sample = s.seq != s.rows && (wanted & (1 << kGate)) != 0;
  const int whole = per_sample ? wanted & ~(1 << kGate) : wanted;
  if (wanted == 0) return OPUS_OK;
  return launch_columns_join(parts, s.blocks, s, whole, out, gates, per_sample ? a.gate_rows : 0, a.grad_gate, st);
}

template <typename TX, typename TY, int V, int Form, bool Bias>
int backward_by_width(const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws, cudaStream_t st) {
  // 16 elements a thread, 8 where the sums of 16 f32 columns would not leave registers enough (with biases) and 8
  // reach the row's end.  Single elements 8: 32768 x 1601 bf16 189 us (16: 224), 16384 x 5001 327 us (506)
  constexpr bool Full = Form != kGradJoin;
  constexpr int kMost = V == 1 ? 8 : narrow_vectors(V, Full), kFewer = fewer_vectors(V, Full);
  constexpr bool kLean = V == 4 && Full && Bias;
  NormShape s;
  if (a.d > kNormThreads * kMost * V) {
    constexpr int kWide = kLean ? kFewer : kMost;
    const int rc = norm_shape_wide(&a, V, kWide, &s);
    return rc ? rc : launch_backward<TX, TY, V, kWide, Form, Bias, true>(s, a, wanted, out, ws, st);
  }
  const bool lean = kLean && a.d <= norm_narrow(V, Full) / 2;
  const int nv = norm_shape(&a, V, lean ? kFewer : kMost, &s);
  if constexpr (V > 1) {
    if (nv == 1) return launch_backward<TX, TY, V, 1, Form, Bias, false>(s, a, wanted, out, ws, st);
  }
  if constexpr (V < 8) {
    if (nv <= kFewer) return launch_backward<TX, TY, V, kFewer, Form, Bias, false>(s, a, wanted, out, ws, st);
  }
  norm_shape(&a, V, kMost, &s, grad_threads(V, kMost, Form, Bias, false));
  return launch_backward<TX, TY, V, kMost, Form, Bias, false>(s, a, wanted, out, ws, st);
}

template <typename TX, typename TY, int V>
int backward_by_form(const opus_residual_norm_args& a, int wanted, const ColumnOutputs& out, uint8_t* ws, cudaStream_t st) {
  const bool bias = a.post_bias != nullptr || (wanted & (1 << kBias)) != 0;
  if (a.gate != nullptr && a.gate_rows > 1)
    return bias ? backward_by_width<TX, TY, V, kGradSamples, true>(a, wanted, out, ws, st)
                : backward_by_width<TX, TY, V, kGradSamples, false>(a, wanted, out, ws, st);
  if (a.post || a.gate != nullptr)
    return bias ? backward_by_width<TX, TY, V, kGradFull, true>(a, wanted, out, ws, st)
                : backward_by_width<TX, TY, V, kGradFull, false>(a, wanted, out, ws, st);
  return bias ? backward_by_width<TX, TY, V, kGradJoin, true>(a, wanted, out, ws, st)
              : backward_by_width<TX, TY, V, kGradJoin, false>(a, wanted, out, ws, st);
}

template <typename TX, typename TY>
int backward_by_alignment(const opus_residual_norm_args& a, bool vec, int wanted, const ColumnOutputs& out, uint8_t* ws,
                        cudaStream_t st) {
  return vec ? backward_by_form<TX, TY, 16 / sizeof(TX)>(a, wanted, out, ws, st)
             : backward_by_form<TX, TY, 1>(a, wanted, out, ws, st);
}

}  // namespace
}  // namespace opus
