// Rows of the residual norm in registers: the parts that its forward and
// backward kernels share.
//
// A row of d elements is held by a group of `group` threads (a power of two up
// to 32, or whole warps), thread t holding the vectors t, t + group, ... of V
// elements each, NV of them, as they are in memory.  Every group owns a run of
// neighbouring rows and loads one while it works on the one before.
//
// What bounds these kernels besides HBM is how many instructions a row takes:
// at 6.5 TB/s an SM has about 2800 issue slots for a forward row of 2048 bf16
// elements.  So 16 elements a thread (each thread's addresses, shuffles and
// barriers serve more of them), parameters as f32 in shared memory with ones
// and zeros where there are none (no branches between loads, which otherwise
// wait for each other), and 16-bit elements taken apart by words.
#pragma once

#include "elements.cuh"

namespace opus {

constexpr int kNormMaxWidth = 16384;

// A block has up to 256 threads of up to 16 elements each (the forward's large blocks 512, one form of the backward
// 384).  Vectors of one element need more registers each
// (an address, a predicate): with a norm of y or a gate they are 8 at most.  Registers that spill cost more than
// anything else here: 50000 x 771 f32 with both norms took 335 us forward with 16 elements a thread and 820 bytes
// spilled, 155 us with 8; without them 128 us with 8, 107 with 16.  Rows wider than a block are split among the
// blocks of a cluster, which have the same registers each and share the row's sums.
constexpr int kNormThreads = 256;
constexpr int kNormMostThreads = 512;
constexpr int narrow_vectors(int V, bool full) { return V == 1 && full ? 8 : 16 / V; }
constexpr int norm_narrow(int V, bool full) { return kNormThreads * narrow_vectors(V, full) * V; }
// the smaller choice for shorter rows (vectors of 8: one vector)
constexpr int fewer_vectors(int V, bool full) { return V == 1 ? 4 : narrow_vectors(V, full) / 2; }

struct NormShape {
  int64_t rows;
  int64_t seq;  // rows that share a row of the gate (rows of a sample); `rows` for one gate
  int d;
  int group, groups;  // threads of a row in a block, rows of a block
  int ranks;          // blocks of a row: 1, or a cluster's (with groups = 1)
  int layer;          // LayerNorm (1) or RMS norm (0)
  float eps;
  int blocks;  // of the launch, or clusters of them
  int* err;    // the device error word (clusters)
};

// The rows [first, last) of worker w among n.
struct RowRun {
  int64_t first, last;
  __device__ RowRun(int64_t rows, int64_t w, int64_t n) {
    const int64_t each = rows / n, more = rows % n;
    first = w * each + (w < more ? w : more);
    last = first + each + (w < more ? 1 : 0);
  }
};

// Shared memory of a group's sums: slots of its warps (a multiple of 4; of every block of the row), twice for two
// values, twice for two turns; two mbarriers behind them for a cluster.
__host__ __device__ constexpr int group_slots(int group) { return group <= 32 ? 0 : ((group >> 5) + 3) / 4 * 4; }
__host__ __device__ constexpr int group_floats(int group, int groups, int ranks) {
  return 4 * groups * ranks * group_slots(group) + (ranks > 1 ? 4 : 0);
}

// Whether a thread's group may be less than a warp (norm_shape's smallest vector counts).
constexpr bool norm_sub_warp(int V, int NV) { return NV == 1 || (V == 1 && NV == 4); }

// Sums over the group of up to two values each, in a fixed order; the result is in every thread of the group.
// A call takes one barrier of the group's own.  The blocks of a cluster send their warps' sums to each other, counted
// on the receiver's mbarrier: a barrier of the cluster would wait for the row's stores to HBM too (8192 x 8192 bf16
// backward with both norms: 340 us, 250 so).
// `turn` alternates between two buffers: a block sends the sums after next only when it has had the next ones of
// every warp, and those are sent after the warp has read the buffer.
template <bool SubWarp, bool Cluster>
struct GroupSum {
  float* buf;
  int slots, span, barrier, threads;
  unsigned lanes;
  int turn;
  const NormShape& shape;
  uint32_t phases;  // bit 0 or 1: the parity that the turn's mbarrier completes next; bit 2: a wait ran out (the sums
                    // are wrong from there, and the error word says so)

  // every thread of the block calls it once
  __device__ GroupSum(float* shared, const NormShape& s)
      : threads(s.group), lanes(0xffffffffu), turn(0), shape(s), phases(0) {
    slots = group_slots(s.group) * (Cluster ? s.ranks : 1);  // of the row's warps, zeros behind each block's
    span = s.groups * slots;
    const int g = static_cast<int>(threadIdx.x) / s.group;
    buf = shared + g * slots;
    static_assert(kNormMostThreads / 64 < 16, "a named barrier, 1 to 15, for each group of more than a warp");
    barrier = 1 + g;
    if (SubWarp && s.group < 32) lanes = ((1u << s.group) - 1) << ((threadIdx.x & 31) / s.group * s.group);
    for (int i = threadIdx.x; i < 4 * span; i += blockDim.x) shared[i] = 0.f;
    if constexpr (Cluster) {
      uint64_t* bars = reinterpret_cast<uint64_t*>(shared + 4 * span);
      if (threadIdx.x == 0) {
        mbar_init(bars, 1);
        mbar_init(bars + 1, 1);
        fence_mbar_init();
      }
      __syncwarp();
      cluster_sync();  // before another block writes here
    } else {
      __syncthreads();
    }
  }
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N], int t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (SubWarp && o >= threads) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(lanes, v[i], o);
    }
    if (slots == 0) return;
    float* b = buf + turn;
    turn = 2 * span - turn;
    if constexpr (Cluster) {
      const int which = turn == 0;  // of the turn that b is
      uint64_t* bar = reinterpret_cast<uint64_t*>(buf + 4 * span) + which;
      const int lane = t & 31;
      if (phases < 4) {
        if (t == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(shape.ranks * (threads >> 5) * N * sizeof(float)));
        if (lane < shape.ranks) {
          float* own = b + cluster_ctarank() * group_slots(threads) + (t >> 5);
#pragma unroll
          for (int i = 0; i < N; ++i) send(own + i * span, bar, lane, v[i]);
        }
        if (!mbar_wait(bar, phases >> which & 1, nullptr, shape.err, kDevTimeoutRow)) phases |= 4;
        phases ^= 1u << which;
      }
      __syncwarp();
    } else {
      if ((t & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i * span + (t >> 5)] = v[i];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(b + i * span);
      float s = (q.x + q.y) + (q.z + q.w);
      for (int w = 4; w < slots; w += 4) {
        const float4 r = *reinterpret_cast<const float4*>(b + i * span + w);
        s += (r.x + r.y) + (r.z + r.w);
      }
      v[i] = s;
    }
  }

  // at the kernel's end, by every thread: no block leaves while another may still send to it
  __device__ __forceinline__ void leave() {
    if constexpr (Cluster) {
      __syncwarp();
      cluster_sync();
    }
  }

 private:
  // *p = v in the shared memory of the cluster's block `peer`, counted on its mbarrier
  static __device__ __forceinline__ void send(float* p, uint64_t* bar, int peer, float v) {
    const uint32_t to = mapa_shared(smem_u32(p), static_cast<uint32_t>(peer));
    const uint32_t on = mapa_shared(smem_u32(bar), static_cast<uint32_t>(peer));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(v), "r"(on)
                 : "memory");
  }
};

// Which columns a thread holds.
template <int V, int NV>
struct Columns {
  int at[NV];
  bool own[NV];
  __device__ Columns(const NormShape& s, int t, int base) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      at[k] = base + (k * s.group + t) * V;
      own[k] = at[k] < s.d;
    }
  }
};

// A thread's part of a row, as it is in memory; zeros beyond the row.
template <typename T, int V, int NV>
struct RawRow {
  Vec<T, V> v[NV];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k].zero();
  }
  __device__ __forceinline__ void load(const T* row, const Columns<V, NV>& c) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (c.own[k]) v[k] = *reinterpret_cast<const Vec<T, V>*>(row + c.at[k]);
  }
  __device__ __forceinline__ void get(float (&r)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k].get(r[k]);
  }
};

template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(T* row, const Columns<V, NV>& c, const float (&r)[NV][V]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (c.own[k]) store_vec<T, V>(row + c.at[k], r[k]);
}

// mean (0 for an RMS norm) and 1 / sqrt(mean square about it + eps) of a row (zeros beyond it)
template <bool Pairs, int V, int NV, typename Sum>
__device__ __forceinline__ float2 row_stats(const float (&r)[NV][V], const NormShape& s, const Columns<V, NV>& c, int t, Sum& sum) {
  const float inv_d = 1.0f / static_cast<float>(s.d);
  float mean = 0.f;
  float q[2] = {0.f, 0.f};  // two chains
  if (s.layer) {
#pragma unroll
    for (int k = 0; k < NV; ++k) vsum<Pairs>(q, r[k]);
    float a[1] = {q[0] + q[1]};
    sum(a, t);
    mean = a[0] * inv_d;
    q[0] = q[1] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const float m = c.own[k] ? mean : 0.f;
    if constexpr (Pairs) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = r[k][i];
      vadd<true>(v, -m);
      vdot<true>(q, v, v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) q[i & 1] = fmaf(r[k][i] - m, r[k][i] - m, q[i & 1]);
    }
  }
  float whole[1] = {q[0] + q[1]};
  sum(whole, t);
  return make_float2(mean, rsqrtf(whole[0] * inv_d + s.eps));
}

// r = (r - mean) / sd of a row with those statistics (an RMS norm's mean is 0)
template <bool Pairs, int V, int NV>
__device__ __forceinline__ void normalize(float (&r)[NV][V], float mean, float rstd) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    vadd<Pairs>(r[k], -mean);
    vmul<Pairs>(r[k], rstd);
  }
}

// V neighbours of an array whose type is known at run time, in accesses of up to 16 bytes (V > 1: aligned arrays).
template <typename T, int V>
__device__ __forceinline__ void load_param_as(const void* p, int64_t at, float (&r)[V]) {
  constexpr int W = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
  for (int j = 0; j < V / W; ++j) {
    float part[W];
    load_vec<T, W>(static_cast<const T*>(p) + at + j * W, part);
#pragma unroll
    for (int i = 0; i < W; ++i) r[j * W + i] = part[i];
  }
}
template <int V>
__device__ __forceinline__ void load_param_vec(const void* p, int dtype, int64_t at, float (&r)[V]) {
  if (dtype == OPUS_DTYPE_F32) load_param_as<float, V>(p, at, r);
  else if (dtype == OPUS_DTYPE_F16) load_param_as<__half, V>(p, at, r);
  else load_param_as<__nv_bfloat16, V>(p, at, r);
}

// A thread's part of one of the parameters' rows, from where it is (`other` where there is none, 0 beyond the row).
// The branches on the type enclose all of a thread's loads.
template <typename T, int NV, int V>
__device__ __forceinline__ void load_param_row_as(const void* p, int64_t at, const Columns<V, NV>& c, float (&r)[NV][V]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (c.own[k]) load_param_as<T, V>(p, at + c.at[k], r[k]);
}
template <int NV, int V>
__device__ __forceinline__ void load_param_row(const void* p, int dtype, int64_t at, float other, const Columns<V, NV>& c,
                                               float (&r)[NV][V]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) r[k][i] = c.own[k] ? other : 0.f;
  if (p == nullptr) return;
  if (dtype == OPUS_DTYPE_F32) load_param_row_as<float>(p, at, c, r);
  else if (dtype == OPUS_DTYPE_F16) load_param_row_as<__half>(p, at, c, r);
  else load_param_row_as<__nv_bfloat16>(p, at, c, r);
}

// A parameter of d elements that rows share, as f32 in shared memory: `other` where there is none and 0 beyond the
// row; vectors of 8 lie in two planes of 4, so that neighbouring lanes read neighbouring 16 bytes.  A block of a
// cluster has the columns from `base`.
template <int NV, int V>
struct Param {
  const void* p;
  int dtype, base;
  float other;
  float *near, *far;  // the two planes
  __device__ __forceinline__ Param(const void* p_, int dtype_, float other_, int base_)
      : p(p_), dtype(dtype_), base(base_), other(other_), near(nullptr), far(nullptr) {}
  static __host__ __device__ int size(int group) { return group * NV * V; }
  // by every thread; a barrier has to follow.  times: another parameter to multiply by, or NULL
  __device__ __forceinline__ void fill(float** shared, const NormShape& s, const void* times = nullptr, int times_dtype = 0) {
    near = *shared;
    const int whole = size(s.group);
    far = near + whole / 2;
    *shared += whole;
    for (int col = threadIdx.x * V; col < whole; col += blockDim.x * V) {
      const bool own = base + col < s.d;
      float r[V];
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = own ? other : 0.f;
      if (p != nullptr && own) load_param_vec<V>(p, dtype, base + col, r);
      if (times != nullptr && own) {
        float m[V];
        load_param_vec<V>(times, times_dtype, base + col, m);
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] *= m[i];
      }
      if constexpr (V == 8) {
        *reinterpret_cast<float4*>(near + col / 2) = make_float4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<float4*>(far + col / 2) = make_float4(r[4], r[5], r[6], r[7]);
      } else {
        store_vec<float, V>(near + col, r);
      }
    }
  }
  __device__ __forceinline__ void row(const Columns<V, NV>& c, float (&r)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = c.at[k] - base;
      if constexpr (V == 8) {
        const float4 a = *reinterpret_cast<const float4*>(near + at / 2);
        const float4 b = *reinterpret_cast<const float4*>(far + at / 2);
        r[k][0] = a.x, r[k][1] = a.y, r[k][2] = a.z, r[k][3] = a.w;
        r[k][4] = b.x, r[k][5] = b.y, r[k][6] = b.z, r[k][7] = b.w;
      } else {
        load_vec<float, V>(near + at, r[k]);
      }
    }
  }
};

// Sets a kernel's dynamic shared memory limit where it needs more than the default.
template <auto Kernel>
int allow_shared(int bytes) {
  if (bytes > 48 * 1024) OPUS_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return OPUS_OK;
}

// Blocks of a kernel that one multiprocessor holds.
template <auto Kernel>
int resident_blocks(int threads, int shared_bytes) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, shared_bytes) != cudaSuccess || n < 1) n = 1;
  return n;
}

// A launch of s.blocks rows' blocks or clusters: as many as the device holds at once and the rows can use, at most
// `cap` blocks a multiprocessor.
struct NormLaunch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute cluster[1];
  int shared;

  template <auto Kernel>
  int plan(NormShape* s, int shared_floats, int cap, cudaStream_t st) {
    const int threads = s->group * s->groups;
    shared = shared_floats * static_cast<int>(sizeof(float));
    const int rc = allow_shared<Kernel>(shared);
    if (rc) return rc;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(shared);
    cfg.stream = st;
    int64_t most;
    if (s->ranks == 1) {
      const int held = resident_blocks<Kernel>(threads, shared);
      most = static_cast<int64_t>(sm_count()) * (held < cap ? held : cap);
    } else {
      cluster[0].id = cudaLaunchAttributeClusterDimension;
      cluster[0].val.clusterDim.x = static_cast<unsigned>(s->ranks);
      cluster[0].val.clusterDim.y = cluster[0].val.clusterDim.z = 1;
      cfg.attrs = cluster;
      cfg.numAttrs = 1;
      cfg.gridDim = dim3(static_cast<unsigned>(s->ranks));
      int held = 0;
      if (cudaOccupancyMaxActiveClusters(&held, Kernel, &cfg) != cudaSuccess || held < 1) held = 1;
      const int64_t bound = static_cast<int64_t>(sm_count()) * cap / s->ranks;
      most = held < bound ? held : bound;
    }
    const int64_t need = (s->rows + s->groups - 1) / s->groups;
    s->blocks = static_cast<int>(need < most ? need : most);
    cfg.gridDim = dim3(static_cast<unsigned>(s->blocks * s->ranks));
    return OPUS_OK;
  }
};

int norm_shape(const opus_residual_norm_args* a, int V, int most, NormShape* s, int threads = kNormThreads);
int norm_shape_wide(const opus_residual_norm_args* a, int V, int NV, NormShape* s);
int check_norm(const char* what, const opus_residual_norm_args* a);
bool norm_params_aligned(const opus_residual_norm_args* a);

// ---- the backward's sums over rows
enum Column : int { kWeight = 0, kBias, kPostWeight, kPostBias, kGate, kColumns };

struct ColumnOutputs {
  void* p[kColumns];
  int dtype[kColumns];
};

inline int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

constexpr int kGradBlocksPerSm = 4;  // of the backward at most: bounds the workspace

// The kernels of one pair of types are compiled in a file of their own (residual_norm_<types>.cu).
#define OPUS_NORM_LAUNCHES(NAME)                                                                                       \
  int residual_norm_##NAME(const opus_residual_norm_args& a, bool vec, cudaStream_t st);                               \
  int residual_norm_grad_##NAME(const opus_residual_norm_args& a, bool vec, int wanted, const ColumnOutputs& out,      \
                                uint8_t* ws, cudaStream_t st);
OPUS_NORM_LAUNCHES(bf16)
OPUS_NORM_LAUNCHES(f16)
OPUS_NORM_LAUNCHES(f32)
OPUS_NORM_LAUNCHES(f32_bf16)
OPUS_NORM_LAUNCHES(f32_f16)
#undef OPUS_NORM_LAUNCHES

}  // namespace opus
