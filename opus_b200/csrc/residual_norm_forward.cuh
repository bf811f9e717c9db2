// Residual norm, forward: kernels and their launch, for one pair of types (included by residual_norm_<types>.cu).
//
//   z = y or N(y) w_post + b_post;  h = r x + g z;  n = N(h) w + b
//
// N(v) = v / sqrt(mean v^2 + eps), or (v - mean) / sqrt(var + eps) with the
// variance summed about the mean (two sums over the registers, so no
// cancellation).  n is the norm of the h that is stored: what the next block
// sees is the norm of the residual stream as the backward will read it.
//
// Bound: HBM bandwidth; x and y are read once, h and n written once, nothing
// else but 16 bytes of statistics a row.  65536 x 2048 bf16: 185 us, 5.8 TB/s;
// 32768 x 2048 f32 185 us, 5.8 TB/s.  With norms on both sides and a gate 181 us,
// 5.9 TB/s: the gate that all rows share is folded into post_weight and
// post_bias once a block, and biases that are not there are not read.  Reading
// all five arrays from shared memory for every row took 213 us, its warps
// waiting for that memory most.  f32: 175 us, 6.1 TB/s, with the gate apart
// (gate_apart).
#pragma once

#include "residual_norm.cuh"

namespace opus {
namespace {

enum Form : int { kAlone, kJoin, kFull };  // no y; y; y with a norm or a gate

// What holds a row: a block (or a group of its threads), a block of twice the threads, which has no parameter sums to
// keep in registers and needs no other block, or the blocks of a cluster, each with a range of the columns.  At 8192
// columns the larger block takes 100 us where a cluster of two takes 109 (8192 rows, bf16, layer norms; 167 and 206 with
// both norms and a gate).
enum Split : int { kBlock, kLargeBlock, kCluster };

// Bias: with a bias or post_bias.  Apart: one gate for all rows, in an array of its own (ones where there is none).
template <typename TX, typename TY, int V, int NV, int F, bool Bias, int By, bool Apart>
__global__ void __launch_bounds__(By == kLargeBlock ? kNormMostThreads : kNormThreads,
                                  By == kLargeBlock ? 1 : F == kFull || V < 8 ? 2 : 3)
    residual_norm_kernel(const __grid_constant__ NormShape s, const __grid_constant__ opus_residual_norm_args a) {
  extern __shared__ __align__(16) float shared[];
  constexpr bool kPairs = V == 8 && F == kFull;
  const int t = threadIdx.x % s.group;
  const int g = threadIdx.x / s.group;
  constexpr bool Wide = By == kCluster;
  const int rank = Wide ? static_cast<int>(cluster_ctarank()) : 0;
  const int base = Wide ? rank * s.group * NV * V : 0;
  const int64_t unit = Wide ? blockIdx.x / s.ranks : blockIdx.x;
  const RowRun run(s.rows, unit * s.groups + g, static_cast<int64_t>(s.blocks) * s.groups);
  const Columns<V, NV> c(s, t, base);
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
  GroupSum<norm_sub_warp(V, NV), Wide> sum(shared, s);
  float* place = shared + group_floats(s.group, s.groups, Wide ? s.ranks : 1);
  Param<NV, V> w(a.weight, a.weight_dtype, 1.f, base), b(a.bias, a.bias_dtype, 0.f, base);
  Param<NV, V> pw(a.post_weight, a.post_weight_dtype, 1.f, base), pb(a.post_bias, a.post_bias_dtype, 0.f, base);
  Param<NV, V> q(a.gate, a.gate_dtype, 1.f, base);
  w.fill(&place, s);
  if constexpr (Bias) b.fill(&place, s);
  const bool one_gate = s.seq == s.rows;  // it is folded into the norm's weight and bias, or apart
  if constexpr (F == kFull) {
    const void* gate = one_gate && !Apart ? a.gate : nullptr;
    pw.fill(&place, s, gate, a.gate_dtype);
    if constexpr (Bias) pb.fill(&place, s, gate, a.gate_dtype);
    if constexpr (Apart) q.fill(&place, s);
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
        ys = row_stats<kPairs>(u, s, c, t, sum);
        normalize<kPairs>(u, ys.x, ys.y);
      }
      pw.row(c, p);
      if constexpr (Bias) {
        float o[NV][V];
        pb.row(c, o);
#pragma unroll
        for (int k = 0; k < NV; ++k) vfma<kPairs>(u[k], p[k], o[k]);
      } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) vmul<kPairs>(u[k], p[k]);
      }
      if (Apart && one_gate) {  // both branches are part of what gate_apart's figures were measured on
        q.row(c, p);
#pragma unroll
        for (int k = 0; k < NV; ++k) vmul<kPairs>(u[k], p[k]);
      }
      if (!one_gate) {
        if (row >= until) {
          gate_at = row / s.seq * s.d;
          until = (row / s.seq + 1) * s.seq;
        }
        load_param_row(a.gate, a.gate_dtype, gate_at, 1.f, c, p);
#pragma unroll
        for (int k = 0; k < NV; ++k) vmul<kPairs>(u[k], p[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (F == kAlone) vmul<kPairs>(h[k], a.residual_scale);
      else vfma<kPairs>(h[k], a.residual_scale, u[k]);
      Vec<TX, V> stored;
      stored.set(h[k]);
      stored.get(h[k]);  // what is normed is what is stored
      if (c.own[k] && (F != kAlone || a.h != nullptr)) *reinterpret_cast<Vec<TX, V>*>(hp + c.at[k]) = stored;
    }
    hp += s.d;
    const float2 hs = row_stats<kPairs>(h, s, c, t, sum);
    w.row(c, u);
    normalize<kPairs>(h, hs.x, hs.y);
    if constexpr (Bias) {
      float o[NV][V];
      b.row(c, o);
#pragma unroll
      for (int k = 0; k < NV; ++k) vfma<kPairs>(h[k], u[k], o[k]);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) vmul<kPairs>(h[k], u[k]);
    }
    store_row(np, c, h);
    np += s.d;
    if (t == 0 && rank == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(hs.x, hs.y, ys.x, ys.y);
  }
  sum.leave();
}

template <typename TX, typename TY, int V, int NV, int F, bool Bias, int By, bool Apart = false>
int launch_forward(NormShape s, const opus_residual_norm_args& a, cudaStream_t st) {
  constexpr auto kernel = residual_norm_kernel<TX, TY, V, NV, F, Bias, By, Apart>;
  const int arrays = (F == kFull ? 2 : 1) * (Bias ? 2 : 1) + (Apart ? 1 : 0);
  NormLaunch launch;
  const int rc = launch.plan<kernel>(&s, group_floats(s.group, s.groups, s.ranks) + arrays * Param<NV, V>::size(s.group), 32, st);
  if (rc) return rc;
  OPUS_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, kernel, s, a));
  note_launch();
  return OPUS_OK;
}

// Whether one gate of f32 streams is kept apart.  Folding it takes a read of shared memory and a multiplication from each
// element, and yet HBM is left less well used where all of a multiprocessor's 16 warps work: the kernel then waits for
// HBM alone, which moves 6.1 to 6.3 TB/s while the read lies between a row's two sums and 5.5 to 5.8 without it.  512 MB
// in and out, folded and apart, without biases: RMS norms of 2048 columns 188 and 174 us, 4096 196 and 176, 1792 187 and
// 172, 768 185 and 176; layer norms of 2048 199 and 172, with biases too; 1024 196 and 175.  Rows that leave warps or
// lanes idle, or lie in one warp, are bound by what they issue: 1280 columns 175 and 192, 640 177 and 195, 5120 180 and
// 216, 512 185 and 191; layer norms or biases also where a row takes the block: 3712 columns 179 and 199.  (Rows
// of five warps would gain apart, 2560 columns 192 and 176, those of six and seven would not.)  A gate
// for each sample is read from where it is: 2048 columns 172 us, 185 in the kernel for one gate.
// With 16-bit blocks only rows of one or two warps without an idle lane come to wait for HBM: 512 columns 144 and 140 us,
// layer norms 147 and 133, with biases 151 and 132; 1024 columns 144 and 132, 147 and 137, but 140 and 142 with biases.
// 960 columns take 141 and 138, layer norms 139 and 146; 768 columns 136 and 152, 2048 139 and 139.
bool gate_apart(const NormShape& s, int slots, bool bias, bool f32_blocks) {
  if (s.seq != s.rows || s.group * s.groups != kNormThreads) return false;
  if (!f32_blocks) return s.d == s.group * slots && s.group <= (bias ? 32 : 64);
  if (s.group <= 32) return false;
  if (!s.layer && !bias) return 4 * s.d >= 3 * s.group * slots;
  return s.groups > 1 && 8 * s.d >= 7 * s.group * slots;
}

template <typename TX, typename TY, int V, int F, bool Bias>
int forward_by_width(const opus_residual_norm_args& a, cudaStream_t st) {
  NormShape s;
  constexpr bool kBoth = F == kFull;
  constexpr int kMost = narrow_vectors(V, kBoth), kFewer = fewer_vectors(V, kBoth);
  if constexpr (V > 1) {  // single elements would need 1024 threads of 64 registers
    static_assert(2 * kNormThreads == kNormMostThreads, "what a large block holds");
    if (a.d > norm_narrow(V, kBoth) && a.d <= 2 * norm_narrow(V, kBoth)) {
      norm_shape(&a, V, kMost, &s);
      return launch_forward<TX, TY, V, kMost, F, Bias, kLargeBlock>(s, a, st);
    }
  }
  if (a.d > norm_narrow(V, kBoth)) {
    const int rc = norm_shape_wide(&a, V, kMost, &s);
    return rc ? rc : launch_forward<TX, TY, V, kMost, F, Bias, kCluster>(s, a, st);
  }
  const int nv = norm_shape(&a, V, kMost, &s);
  if constexpr (V > 1) {
    if (nv == 1) return launch_forward<TX, TY, V, 1, F, Bias, kBlock>(s, a, st);
  }
  if constexpr (V < 8) {
    if (nv <= kFewer) return launch_forward<TX, TY, V, kFewer, F, Bias, kBlock>(s, a, st);
  }
  if constexpr (V == 4 && kBoth) {
    if (gate_apart(s, V * kMost, Bias, sizeof(TY) == 4)) return launch_forward<TX, TY, V, kMost, F, Bias, kBlock, true>(s, a, st);
  }
  return launch_forward<TX, TY, V, kMost, F, Bias, kBlock>(s, a, st);
}

template <typename TX, typename TY, int V, int F>
int forward_by_bias(const opus_residual_norm_args& a, cudaStream_t st) {
  return a.bias != nullptr || a.post_bias != nullptr ? forward_by_width<TX, TY, V, F, true>(a, st)
                                                     : forward_by_width<TX, TY, V, F, false>(a, st);
}

template <typename TX, typename TY, int V>
int forward_by_form(const opus_residual_norm_args& a, cudaStream_t st) {
  if (a.post || a.gate != nullptr) return forward_by_bias<TX, TY, V, kFull>(a, st);
  if (a.y != nullptr) return forward_by_bias<TX, TY, V, kJoin>(a, st);
  return forward_by_bias<TX, TY, V, kAlone>(a, st);
}

template <typename TX, typename TY>
int forward_by_alignment(const opus_residual_norm_args& a, bool vec, cudaStream_t st) {
  return vec ? forward_by_form<TX, TY, 16 / sizeof(TX)>(a, st) : forward_by_form<TX, TY, 1>(a, st);
}

}  // namespace
}  // namespace opus
