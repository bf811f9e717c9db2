// Global gradient norm over many tensors, and clipping by it.
//
//   opus_grad_norm    |g| = sqrt(sum_j sum_i g_ji^2), or max_ji |g_ji|
//   opus_clip_grads   the same, then out_j = c g_j with c = min(1, max_norm / (|g| + 1e-6))
//   opus_scale_grads  the second half alone, for a norm that the caller has (joined over ranks, say)
//
// Mathematics.  A thread sums the squares of the up to 32 elements of one
// round of loads in f32 and adds the result to a double, so the rounding error
// of the whole is that of 32 f32 additions however long the list is.  Where
// such a partial sum leaves [1e-25, 1e30] (squares that overflow, or vanish,
// in f32) the same registers are summed again in double.  Partial sums meet in
// a fixed order: the norm is the same for every run on one device.
//
// Bound: HBM bandwidth, reads once for the norm and once more (with the
// writes) to scale; a list of one type below the bound is not written at all
// in place, since c = 1 would write what is there.  292 tensors of 355M f32
// elements within the bound: 206 us, 6.9 TB/s.  580 tensors of 1.56G bf16
// elements clipped: 1525 us, 6.1 TB/s over the three passes (the second read
// is of more than L2 holds); 148 of 124M bf16 into f32: 177 us.  48 small
// tensors: two launches, 18 us a call.
//
// Layout: the list travels as a kernel parameter (addresses, lengths, types:
// no copy to the device, and a captured graph holds its own).  Tensors are cut
// into units of 2048 elements and every block takes one run of neighbouring
// units, so blocks share the elements evenly and look a tensor up once.  The
// scaling launch walks each block's run backwards: what the norm read last is
// still in L2.
#include <algorithm>
#include <new>
#include <vector>

#include "elements.cuh"

namespace opus {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 8;
constexpr int64_t kUnit = 2048;   // elements
constexpr float kNormEps = 1e-6f;  // as torch.nn.utils.clip_grad_norm_ has it

// The tensors of one launch.  Most is 960 for long lists (below the 32764 bytes of parameters) and 64 for
// short ones.
template <int Most>
struct GradTable {
  const void* in[Most];
  void* out[Most];
  int64_t n[Most];
  int64_t first[Most];  // number of the tensor's first unit
  uint8_t types[Most];  // type in | type out << 4
  int count;
  int in_place;  // every out is its in
  int64_t units;
};
constexpr int kShort = 64, kLong = 960;
static_assert(sizeof(GradTable<kLong>) <= 32000, "kernel parameters");

template <int Most>
__device__ __forceinline__ int find_tensor(const GradTable<Most>& t, int64_t unit) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= unit) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// This block's run of units: [*a, *b).
__device__ __forceinline__ void block_run(int64_t units, int64_t* a, int64_t* b) {
  const int64_t each = units / gridDim.x, more = units % gridDim.x, k = blockIdx.x;
  *a = k * each + (k < more ? k : more);
  *b = *a + each + (k < more ? 1 : 0);
}

// Sum (kind 2) or maximum (kind 0: the infinity norm, NaN wins) of doubles.
__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind == 2) return a + b;
  return (a != a || a > b) ? a : b;
}

// Every thread's value joined over the block, in a fixed order; valid in all threads.
__device__ double block_join(double v, int kind) {
  __shared__ double warp_part[kThreads / 32];
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_down_sync(0xffffffffu, v, o), kind);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = warp_part[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) s = join(s, warp_part[w], kind);
  return s;
}

// What one group of elements adds to a thread's partial sum.
template <int N>
__device__ __forceinline__ double group_part(const float (&x)[N], int kind) {
  if (kind != 2) {
    double m = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = join(m, static_cast<double>(fabsf(x[i])), 0);
    return m;
  }
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) s[i & 3] = fmaf(x[i], x[i], s[i & 3]);
  const float f = (s[0] + s[1]) + (s[2] + s[3]);
  if (f > 1e-25f && f < 1e30f) return static_cast<double>(f);
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) d = fma(static_cast<double>(x[i]), static_cast<double>(x[i]), d);
  return d;
}

template <typename T>
__device__ double run_part(const T* p, int64_t n, int kind) {
  constexpr int V = 16 / sizeof(T);
  constexpr int U = 4;
  double acc = 0.0;
  int64_t head = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
  head = head < n ? head : n;
  const int64_t vecs = (n - head) / V;
  const T* body = p + head;
  for (int64_t b = threadIdx.x; b < vecs; b += kThreads * U) {
    float x[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float r[V];
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = 0.f;
      if (b + u * kThreads < vecs) load_vec<T, V>(body + (b + u * kThreads) * V, r);
#pragma unroll
      for (int i = 0; i < V; ++i) x[u * V + i] = r[i];
    }
    acc = join(acc, group_part(x, kind), kind);
  }
  // the up to V - 1 elements before the first 16-byte boundary and after the last
  const int64_t tail = head + vecs * V;
  const int64_t i = threadIdx.x;
  const int64_t at = i < head ? i : tail + (i - head);
  if (at < n) {
    const float x[1] = {to_f32(p[at])};
    acc = join(acc, group_part(x, kind), kind);
  }
  return acc;
}

template <int Most>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ GradTable<Most> t, int kind,
                                                        double* __restrict__ partial) {
  double acc = 0.0;
  int64_t u, last;
  block_run(t.units, &u, &last);
  for (int j = find_tensor(t, u); u < last; ++j) {
    const int64_t stop = j + 1 < t.count && t.first[j + 1] < last ? t.first[j + 1] : last;
    const int64_t at = (u - t.first[j]) * kUnit;
    const int64_t n = t.n[j] - at < (stop - u) * kUnit ? t.n[j] - at : (stop - u) * kUnit;
    const int type = t.types[j] & 15;
    double d;
    if (type == OPUS_DTYPE_F32) d = run_part(static_cast<const float*>(t.in[j]) + at, n, kind);
    else if (type == OPUS_DTYPE_F16) d = run_part(static_cast<const __half*>(t.in[j]) + at, n, kind);
    else d = run_part(static_cast<const __nv_bfloat16*>(t.in[j]) + at, n, kind);
    acc = join(acc, d, kind);
    u = stop;
  }
  acc = block_join(acc, kind);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The norm from the blocks' partial sums: every block of the launch does the
// same additions in the same order.
__device__ float whole_norm(const double* __restrict__ partial, int parts, int kind) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s = join(s, partial[i], kind);
  s = block_join(s, kind);
  return static_cast<float>(kind == 2 ? sqrt(s) : s);
}

__global__ void __launch_bounds__(kThreads) norm_join_kernel(const double* __restrict__ partial, int parts, int kind,
                                                             float* __restrict__ norm) {
  wait_for_predecessors();
  const float n = whole_norm(partial, parts, kind);
  if (threadIdx.x == 0) *norm = n;
}

// From the run's end to its start.
template <typename TI, typename TO>
__device__ void run_scale(const TI* p, TO* q, int64_t n, float c) {
  constexpr int V = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
  constexpr int U = 64 / (V * sizeof(TI));  // 64 bytes of loads a thread in flight
  constexpr uintptr_t in_mask = V * sizeof(TI) - 1, out_mask = V * sizeof(TO) - 1;
  int64_t head = static_cast<int64_t>((V * sizeof(TI) - (reinterpret_cast<uintptr_t>(p) & in_mask)) & in_mask) /
                 static_cast<int>(sizeof(TI));
  head = head < n ? head : n;
  // both sides reach their boundaries together, or the run goes element by element
  if ((reinterpret_cast<uintptr_t>(q + head) & out_mask) != 0) head = n;
  const int64_t vecs = (n - head) / V;
  const int64_t tail = head + vecs * V;
  for (int64_t i = threadIdx.x; i < head + (n - tail); i += kThreads) {
    const int64_t at = i < head ? i : tail + (i - head);
    q[at] = from_f32<TO>(to_f32(p[at]) * c);
  }
  for (int64_t b = vecs - 1 - threadIdx.x; b >= 0; b -= kThreads * U) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b - u * kThreads >= 0) load_vec<TI, V>(p + head + (b - u * kThreads) * V, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b - u * kThreads >= 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] *= c;
        store_vec<TO, V>(q + head + (b - u * kThreads) * V, x[u]);
      }
  }
}

// parts > 0: the norm is joined from partial sums here (and block 0 writes it); otherwise it is read.
template <typename TI, typename TO, int Most>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ GradTable<Most> t, int kind,
                                                         const double* __restrict__ partial, int parts,
                                                         float max_norm, float* __restrict__ norm) {
  wait_for_predecessors();
  float n;
  if (parts > 0) {
    n = whole_norm(partial, parts, kind);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  } else {
    n = *norm;
  }
  float c = max_norm / (n + kNormEps);
  c = c > 1.0f ? 1.0f : c;  // a NaN stays
  if (c == 1.0f && t.in_place) return;
  int64_t first, u;
  block_run(t.units, &first, &u);
  for (int j = find_tensor(t, u - 1); u > first; --j) {
    const int64_t from = t.first[j] > first ? t.first[j] : first;
    const int64_t at = (from - t.first[j]) * kUnit;
    const int64_t len = t.n[j] - at < (u - from) * kUnit ? t.n[j] - at : (u - from) * kUnit;
    run_scale(static_cast<const TI*>(t.in[j]) + at, static_cast<TO*>(t.out[j]) + at, len, c);
    u = from;
  }
}

struct Lists {
  const void* const* in;
  void* const* out;
  const int64_t* n;
  const int* in_types;
  const int* out_types;
  int count;
};

constexpr int64_t kMostElements = int64_t{1} << 48;

int check_lists(const char* what, const Lists& l, bool outs) {
  if (l.count < 0) return set_error(OPUS_ERR_INVALID, "%s: %d tensors", what, l.count);
  if (l.count > 0 && (!l.in || !l.n || !l.in_types || (outs && (!l.out || !l.out_types))))
    return set_error(OPUS_ERR_INVALID, "%s: NULL list", what);
  int64_t whole = 0;
  for (int i = 0; i < l.count; ++i) {
    if (l.n[i] < 0) return set_error(OPUS_ERR_INVALID, "%s: tensor %d has %lld elements", what, i, (long long)l.n[i]);
    if (!dtype_ok(l.in_types[i]) || (outs && !dtype_ok(l.out_types[i])))
      return set_error(OPUS_ERR_UNSUPPORTED, "%s: tensor %d is neither bf16, f16 nor f32", what, i);
    if (l.n[i] > 0 && (!l.in[i] || (outs && !l.out[i])))
      return set_error(OPUS_ERR_INVALID, "%s: tensor %d is NULL", what, i);
    if (reinterpret_cast<uintptr_t>(l.in[i]) % dtype_bytes(l.in_types[i]) != 0 ||
        (outs && reinterpret_cast<uintptr_t>(l.out[i]) % dtype_bytes(l.out_types[i]) != 0))
      return set_error(OPUS_ERR_INVALID, "%s: tensor %d is not aligned to its elements", what, i);
    if (l.n[i] <= kMostElements) whole += l.n[i];
    if (l.n[i] > kMostElements || whole > kMostElements)
      return set_error(OPUS_ERR_UNSUPPORTED, "%s: the list is too long", what);
  }
  return OPUS_OK;
}

// Refuses a list that writes an element twice or writes what it reads elsewhere (outs[j] == grads[j] aside); the norm,
// which every block reads, counts among what is read, or among what is written.
int check_overlap(const char* what, const Lists& l, const float* norm, bool norm_written) {
  struct Range {
    uintptr_t start, end;
    bool written;
  };
  try {
    std::vector<Range> r;
    r.reserve(2 * static_cast<size_t>(l.count) + 1);
    const uintptr_t at = reinterpret_cast<uintptr_t>(norm);
    if (norm != nullptr) r.push_back({at, at + sizeof(float), norm_written});
    for (int i = 0; i < l.count; ++i) {
      if (l.n[i] == 0) continue;
      const uintptr_t in = reinterpret_cast<uintptr_t>(l.in[i]), out = reinterpret_cast<uintptr_t>(l.out[i]);
      const bool in_place = in == out && l.in_types[i] == l.out_types[i];
      if (!in_place) r.push_back({in, in + l.n[i] * dtype_bytes(l.in_types[i]), false});
      r.push_back({out, out + l.n[i] * dtype_bytes(l.out_types[i]), true});
    }
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.start < b.start; });
    uintptr_t read = 0, written = 0;  // how far the ranges so far reach
    for (const Range& x : r) {
      if (x.start < written || (x.written && x.start < read))
        return set_error(OPUS_ERR_INVALID, "%s: an element would be written twice, or written and read elsewhere "
                         "(a tensor listed twice, overlapping views, or outputs or a norm that overlap the inputs)", what);
      uintptr_t& reach = x.written ? written : read;
      reach = x.end > reach ? x.end : reach;
    }
  } catch (const std::bad_alloc&) {
    return set_error(OPUS_ERR_INVALID, "%s: no host memory for %d tensors", what, l.count);
  }
  return OPUS_OK;
}

// Tensors [at, ...) of the list as one launch's table, those of one pair of types when asked for; returns
// the index of the first that did not fit.
template <int Most>
int fill_table(const Lists& l, int at, int types, GradTable<Most>* t) {
  t->count = 0;
  t->in_place = 1;
  t->units = 0;
  for (; at < l.count && t->count < Most; ++at) {
    const int pair = l.in_types[at] | (l.out ? l.out_types[at] << 4 : 0);
    if (l.n[at] == 0 || (types >= 0 && types != pair)) continue;
    const int k = t->count++;
    t->in[k] = l.in[at];
    t->out[k] = l.out ? l.out[at] : nullptr;
    t->in_place &= t->in[k] == t->out[k];
    t->n[k] = l.n[at];
    t->first[k] = t->units;
    t->types[k] = static_cast<uint8_t>(pair);
    t->units += (l.n[at] + kUnit - 1) / kUnit;
  }
  return at;
}

int grid_of(int64_t units) {
  const int64_t most = static_cast<int64_t>(sm_count()) * kBlocksPerSm;
  return static_cast<int>(units < most ? units : most);
}

// Partial sums of every launch side by side; *parts is their number.
template <int Most>
int launch_norm(const Lists& l, int kind, double* partial, int* parts, cudaStream_t st) {
  GradTable<Most> t;
  *parts = 0;
  for (int at = 0; at < l.count;) {
    at = fill_table(l, at, -1, &t);
    if (t.units == 0) continue;
    const int grid = grid_of(t.units);
    norm_kernel<Most><<<grid, kThreads, 0, st>>>(t, kind, partial + *parts);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    *parts += grid;
  }
  return OPUS_OK;
}

template <typename TI, typename TO, int Most>
int launch_scale_pair(const Lists& l, int types, int kind, const double* partial, int parts, float max_norm,
                      float* norm, cudaStream_t st) {
  GradTable<Most> t;
  for (int at = 0; at < l.count;) {
    at = fill_table(l, at, types, &t);
    if (t.units == 0) continue;
    OPUS_CUDA_TRY(launch_early(scale_kernel<TI, TO, Most>, dim3(grid_of(t.units)), kThreads, 0, st, t, kind, partial,
                               parts, max_norm, norm));
    note_launch();
  }
  return OPUS_OK;
}

// One launch for each pair of types in the list (a kernel of all nine pairs takes 238 registers and ran at a
// quarter of the bandwidth).
template <int Most>
int launch_scale_most(const Lists& l, int kind, const double* partial, int parts, float max_norm, float* norm,
                      cudaStream_t st) {
  unsigned seen[3] = {0, 0, 0};
  for (int i = 0; i < l.count; ++i)
    if (l.n[i] > 0) seen[l.in_types[i]] |= 1u << l.out_types[i];
  int rc = OPUS_OK;
#define OPUS_SCALE_PAIR(A, TA, B, TB)          \
  if (rc == OPUS_OK && (seen[A] & (1u << B)))  \
    rc = launch_scale_pair<TA, TB, Most>(l, A | B << 4, kind, partial, parts, max_norm, norm, st)
  OPUS_SCALE_PAIR(OPUS_DTYPE_BF16, __nv_bfloat16, OPUS_DTYPE_BF16, __nv_bfloat16);
  OPUS_SCALE_PAIR(OPUS_DTYPE_BF16, __nv_bfloat16, OPUS_DTYPE_F32, float);
  OPUS_SCALE_PAIR(OPUS_DTYPE_BF16, __nv_bfloat16, OPUS_DTYPE_F16, __half);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F32, float, OPUS_DTYPE_BF16, __nv_bfloat16);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F32, float, OPUS_DTYPE_F32, float);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F32, float, OPUS_DTYPE_F16, __half);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F16, __half, OPUS_DTYPE_BF16, __nv_bfloat16);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F16, __half, OPUS_DTYPE_F32, float);
  OPUS_SCALE_PAIR(OPUS_DTYPE_F16, __half, OPUS_DTYPE_F16, __half);
#undef OPUS_SCALE_PAIR
  return rc;
}

int launch_norm(const Lists& l, int kind, double* partial, int* parts, cudaStream_t st) {
  return l.count <= kShort ? launch_norm<kShort>(l, kind, partial, parts, st)
                           : launch_norm<kLong>(l, kind, partial, parts, st);
}

int launch_scale(const Lists& l, int kind, const double* partial, int parts, float max_norm, float* norm,
                 cudaStream_t st) {
  return l.count <= kShort ? launch_scale_most<kShort>(l, kind, partial, parts, max_norm, norm, st)
                           : launch_scale_most<kLong>(l, kind, partial, parts, max_norm, norm, st);
}

int launch_join(const double* partial, int parts, int kind, float* norm, cudaStream_t st) {
  OPUS_CUDA_TRY(launch_early(norm_join_kernel, dim3(1), kThreads, 0, st, partial, parts, kind, norm));
  note_launch();
  return OPUS_OK;
}

int check_norm_args(const char* what, int kind, const void* workspace, int64_t bytes, int count, const float* norm) {
  if (kind != 2 && kind != 0) return set_error(OPUS_ERR_INVALID, "%s: norm kind %d is neither 2 nor 0 (infinity)", what, kind);
  if (!workspace || !norm) return set_error(OPUS_ERR_INVALID, "%s: NULL pointer", what);
  const int64_t need = opus_grad_norm_workspace_bytes(count);
  if (bytes < need)
    return set_error(OPUS_ERR_INVALID, "%s: workspace of %lld bytes, need %lld", what, (long long)bytes, (long long)need);
  if ((reinterpret_cast<uintptr_t>(workspace) & 7) != 0)
    return set_error(OPUS_ERR_INVALID, "%s: workspace must be 8-byte aligned", what);
  return OPUS_OK;
}

}  // namespace
}  // namespace opus

using namespace opus;

extern "C" int64_t opus_grad_norm_workspace_bytes(int count) {
  const int64_t launches = count > kLong ? (count + kLong - 1) / kLong : 1;
  return launches * sm_count() * kBlocksPerSm * 8;
}

extern "C" int opus_grad_norm(const void* const* grads, const int64_t* numels, const int* dtypes, int count,
                              int norm_kind, void* workspace, int64_t workspace_bytes, float* norm, void* stream) {
  const Lists l{grads, nullptr, numels, dtypes, nullptr, count};
  int rc = check_lists("grad_norm", l, false);
  if (rc) return rc;
  rc = check_norm_args("grad_norm", norm_kind, workspace, workspace_bytes, count, norm);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int parts = 0;
  rc = launch_norm(l, norm_kind, partial, &parts, st);
  if (rc) return rc;
  return launch_join(partial, parts, norm_kind, norm, st);
}

extern "C" int opus_scale_grads(const void* const* grads, const int* dtypes, void* const* outs, const int* out_dtypes,
                                const int64_t* numels, int count, float max_norm, const float* norm, void* stream) {
  const Lists l{grads, outs, numels, dtypes, out_dtypes, count};
  int rc = check_lists("scale_grads", l, true);
  if (rc == OPUS_OK) rc = check_overlap("scale_grads", l, norm, false);
  if (rc) return rc;
  if (!norm) return set_error(OPUS_ERR_INVALID, "scale_grads: NULL pointer");
  return launch_scale(l, 2, nullptr, 0, max_norm, const_cast<float*>(norm), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int opus_clip_grads(const void* const* grads, const int* dtypes, void* const* outs, const int* out_dtypes,
                               const int64_t* numels, int count, int norm_kind, float max_norm, void* workspace,
                               int64_t workspace_bytes, float* norm, void* stream) {
  const Lists l{grads, outs, numels, dtypes, out_dtypes, count};
  int rc = check_lists("clip_grads", l, true);
  if (rc == OPUS_OK) rc = check_overlap("clip_grads", l, norm, true);
  if (rc) return rc;
  rc = check_norm_args("clip_grads", norm_kind, workspace, workspace_bytes, count, norm);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int parts = 0;
  rc = launch_norm(l, norm_kind, partial, &parts, st);
  if (rc) return rc;
  if (parts == 0) return launch_join(partial, 0, norm_kind, norm, st);
  return launch_scale(l, norm_kind, partial, parts, max_norm, norm, st);
}
