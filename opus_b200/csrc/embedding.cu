// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   opus_embedding       Y[i] = s W[t_i]
//   opus_embedding_grad  dW[v] (+)= s sum_{i: t_i = v} dY[i]
//
// The gradient.  Positions are sorted by their token (a stable radix sort, so
// equal tokens keep the order of their positions) and the sorted list is cut
// into units of 32 positions.  A warp sums a unit's rows for a slab of columns
// in f32, one run of equal tokens after another, and writes a run that lies
// inside the unit straight into dW.  A run that crosses units leaves its parts
// in a workspace, and a second kernel joins them in order.  No atomics: every
// sum has one order, and the result is the same for every call.
//
// Tokens outside [0, V) give a row of zeros, add to no gradient, and are
// recorded in the device error word.  Tokens equal to padding_idx add to no
// gradient.
//
// Bound: HBM bandwidth; dY is read once (whole rows, in sorted order) and dW
// written once.
#include "elements.cuh"

namespace opus {
namespace {

constexpr int kFwdThreads = 256;

__device__ __forceinline__ int64_t load_token(const void* tokens, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(tokens)[i] : static_cast<const int32_t*>(tokens)[i];
}

template <typename T, int V>
__global__ void __launch_bounds__(kFwdThreads) lookup_kernel(const void* __restrict__ tokens, int wide, int64_t n,
                                                             const T* __restrict__ w, int64_t vocab, int64_t stride,
                                                             int d, float scale, T* __restrict__ y, int* err) {
  const int per_row = d / V;
  const int64_t total = n * per_row;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kFwdThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kFwdThreads) {
    const int64_t row = i / per_row;
    const int col = static_cast<int>(i - row * per_row) * V;
    const int64_t t = load_token(tokens, wide, row);
    float x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = 0.f;
    if (t >= 0 && t < vocab) {
      load_vec<T, V>(w + t * stride + col, x);
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] *= scale;
    } else if (col == 0) {
      record_device_error(err, kDevBadToken);
    }
    store_vec<T, V>(y + row * d + col, x);
  }
}

// ------------------------------------------------------------------ sorting
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 8;                          // keys of a thread
constexpr int kTile = kSortThreads * kSortRounds;       // keys of a block
constexpr int kMaxBits = 9;                             // of a digit
constexpr int kMaxBins = 1 << kMaxBits;

// The sort key of position i: its token, or V (behind every token) for one that adds to no row.
struct KeySource {
  const void* tokens;  // first pass; later passes read keys
  const uint32_t* keys;
  const uint32_t* pos;
  int wide;
  int64_t vocab;
  int64_t padding;
};

__device__ __forceinline__ uint32_t load_key(const KeySource& s, int64_t i, int* err) {
  if (s.keys != nullptr) return s.keys[i];
  const int64_t t = load_token(s.tokens, s.wide, i);
  if (t < 0 || t >= s.vocab) {
    record_device_error(err, kDevBadToken);
    return static_cast<uint32_t>(s.vocab);
  }
  return static_cast<uint32_t>(t == s.padding ? s.vocab : t);
}

// counts[bin * tiles + tile]: keys of the tile whose digit is bin.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(KeySource src, int64_t n, int shift, int bits,
                                                                  int tiles, uint32_t* __restrict__ counts, int* err) {
  __shared__ uint32_t hist[kMaxBins];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(load_key(src, i, err) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) counts[static_cast<int64_t>(b) * tiles + blockIdx.x] = hist[b];
}

// Exclusive prefix sums of `count` values in place, by one block.
constexpr int kScanThreads = 1024;
__global__ void __launch_bounds__(kScanThreads) sort_scan_kernel(uint32_t* __restrict__ counts, int64_t count) {
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int64_t at = 0; at < count; at += kScanThreads * 4) {
    const int64_t i = at + threadIdx.x * 4;
    uint32_t v[4], own = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = i + k < count ? counts[i + k] : 0u;
      own += v[k];
    }
    uint32_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    uint32_t before = carry, whole = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_sum[w];
      whole += warp_sum[w];
    }
    uint32_t run = before + incl - own;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k < count) counts[i + k] = run;
      run += v[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) carry += whole;
    __syncthreads();
  }
}

// Writes every key of the tile, with its position, to its place by this digit.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(KeySource src, int64_t n, int shift, int bits,
                                                                  int tiles, const uint32_t* __restrict__ offsets,
                                                                  uint32_t* __restrict__ keys_out,
                                                                  uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t count[kSortWarps][kMaxBins];
  const int bins = 1 << bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
  __syncthreads();
  // a warp's keys are kSortRounds runs of 32 neighbours: rounds in order keep equal keys in order
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile + warp * (32 * kSortRounds) + lane;
  uint32_t key[kSortRounds], place[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * 32;
    const bool live = i < n;
    key[r] = live ? load_key(src, i, nullptr) : 0u;
    const uint32_t digit = live ? (key[r] >> shift) & (bins - 1) : kMaxBins;
    const uint32_t same = __match_any_sync(0xffffffffu, digit);
    const int leader = __ffs(same) - 1;
    uint32_t before = 0;
    if (live && lane == leader) {
      before = count[warp][digit];
      count[warp][digit] = before + __popc(same);
    }
    before = __shfl_sync(0xffffffffu, before, leader);
    place[r] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    uint32_t at = offsets[static_cast<int64_t>(b) * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = count[w][b];
      count[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * 32;
    if (i >= n) continue;
    const uint32_t at = count[warp][(key[r] >> shift) & (bins - 1)] + place[r];
    keys_out[at] = key[r];
    pos_out[at] = src.pos != nullptr ? src.pos[i] : static_cast<uint32_t>(i);
  }
}

// ------------------------------------------------------------------ sums
constexpr int kUnit = 32;         // sorted positions of a unit
constexpr int kSumWarps = 4;      // units of a block

template <typename TO, int V>
__device__ __forceinline__ void write_row(TO* out, const float (&acc)[V], float scale, int accumulate) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = acc[k] * scale;
  if (accumulate) {
    float o[V];
    load_vec<TO, V>(out, o);
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] += o[k];
  }
  store_vec<TO, V>(out, r);
}

// One warp: one unit, 32 * V columns.  parts[unit]: [0] the part of a run that came from the unit before (or
// fills the unit), [1] the part of a run that starts here and goes on.
template <typename T, typename TO, int V>
__global__ void __launch_bounds__(kSumWarps * 32) sum_kernel(const uint32_t* __restrict__ keys,
                                                             const uint32_t* __restrict__ pos, int64_t n,
                                                             uint32_t vocab, const T* __restrict__ dy, int64_t stride,
                                                             int d, float scale, int accumulate,
                                                             TO* __restrict__ dw, float* __restrict__ parts) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
  const int64_t first = unit * kUnit;
  if (first >= n) return;
  const int col = (blockIdx.y * 32 + lane) * V;
  const bool live = col < d;
  const int64_t mine = first + lane;
  const uint32_t my_key = mine < n ? keys[mine] : vocab;
  const uint32_t my_pos = mine < n ? pos[mine] : 0u;
  const uint32_t before = first > 0 ? keys[first - 1] : vocab;
  const uint32_t after = first + kUnit < n ? keys[first + kUnit] : vocab;
  const int len = __popc(__ballot_sync(0xffffffffu, my_key < vocab));  // keys equal to vocab sort last
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.f;
  bool crossed = false;
  for (int j = 0; j < len; ++j) {
    const uint32_t key = __shfl_sync(0xffffffffu, my_key, j);
    const uint32_t p = __shfl_sync(0xffffffffu, my_pos, j);
    if (j == 0) crossed = before == key;
    float x[V];
    if (live) {
      load_vec<T, V>(dy + static_cast<int64_t>(p) * stride + col, x);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += x[k];
    }
    const uint32_t next = j + 1 < kUnit ? __shfl_sync(0xffffffffu, my_key, j + 1 < kUnit ? j + 1 : 31) : after;
    if (next != key || j + 1 == kUnit) {
      const bool goes_on = j + 1 == kUnit && next == key;
      if (live) {
        if (crossed) store_vec<float, V>(parts + (unit * 2) * d + col, acc);
        else if (goes_on) store_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
        else write_row<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc, scale, accumulate);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] = 0.f;
      crossed = false;
    }
  }
}

// Joins the parts of the run that starts in unit blockIdx.x and goes on behind it, if there is one.
constexpr int kJoinWarps = 8;
template <typename TO, int V>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                               uint32_t vocab, int d, float scale, int accumulate,
                                                               TO* __restrict__ dw, const float* __restrict__ parts) {
  __shared__ float slice[kJoinWarps][32 * V];
  const int64_t unit = blockIdx.x;
  const int64_t end = (unit + 1) * kUnit;
  if (end >= n) return;
  const uint32_t key = keys[end - 1];
  if (key >= vocab || keys[end] != key) return;
  if (unit > 0 && keys[unit * kUnit] == key && keys[unit * kUnit - 1] == key) return;  // it started before
  // the run's last position by bisection
  int64_t lo = end, hi = n - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (keys[mid] == key) lo = mid;
    else hi = mid - 1;
  }
  const int64_t units = lo / kUnit - unit;  // units behind this one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * V;
  const int64_t a = units * warp / kJoinWarps, b = units * (warp + 1) / kJoinWarps;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.f;
  if (col < d) {
    if (warp == 0) load_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
#pragma unroll 4
    for (int64_t u = unit + 1 + a; u < unit + 1 + b; ++u) {
      float x[V];
      load_vec<float, V>(parts + (u * 2) * d + col, x);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += x[k];
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) slice[warp][lane * V + k] = acc[k];
  __syncthreads();
  if (warp == 0 && col < d) {
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += slice[w][lane * V + k];
    write_row<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc, scale, accumulate);
  }
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int bits, passes, digit;
  int64_t tiles, units;
  int64_t keys, counts, parts, bytes;  // offsets of the second keys (two pairs of n), counts, parts; the whole
};

Plan plan_of(int64_t n, int64_t vocab, int d) {
  Plan p{};
  while ((vocab >> p.bits) != 0) ++p.bits;  // the key V itself is used
  p.passes = (p.bits + kMaxBits - 1) / kMaxBits;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.tiles = (n + kTile - 1) / kTile;
  p.units = (n + kUnit - 1) / kUnit;
  p.keys = align256(n * 4);
  p.counts = 4 * p.keys;
  p.parts = p.counts + align256((p.tiles << p.digit) * 4);
  p.bytes = p.parts + align256(p.units * 2 * d * 4);
  return p;
}

template <typename T, typename TO, int V>
int launch_sums(const uint32_t* keys, const uint32_t* pos, const Plan& p, int64_t n, int64_t vocab, const void* dy,
                int64_t stride, int d, float scale, int accumulate, void* dw, float* parts, cudaStream_t st) {
  const unsigned slabs = (d / V + 31) / 32;
  const dim3 grid(static_cast<unsigned>((p.units + kSumWarps - 1) / kSumWarps), slabs);
  sum_kernel<T, TO, V><<<grid, kSumWarps * 32, 0, st>>>(keys, pos, n, static_cast<uint32_t>(vocab),
                                                        static_cast<const T*>(dy), stride, d, scale, accumulate,
                                                        static_cast<TO*>(dw), parts);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  join_kernel<TO, V><<<dim3(static_cast<unsigned>(p.units), slabs), kJoinWarps * 32, 0, st>>>(
      keys, n, static_cast<uint32_t>(vocab), d, scale, accumulate, static_cast<TO*>(dw), parts);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename T, typename TO>
int launch_sums_by_width(bool wide, const uint32_t* keys, const uint32_t* pos, const Plan& p, int64_t n, int64_t vocab,
                         const void* dy, int64_t stride, int d, float scale, int accumulate, void* dw, float* parts,
                         cudaStream_t st) {
  constexpr int V = 16 / (sizeof(T) > sizeof(TO) ? sizeof(T) : sizeof(TO));
  if (wide) return launch_sums<T, TO, V>(keys, pos, p, n, vocab, dy, stride, d, scale, accumulate, dw, parts, st);
  return launch_sums<T, TO, 1>(keys, pos, p, n, vocab, dy, stride, d, scale, accumulate, dw, parts, st);
}

template <typename T>
int launch_lookup(const void* tokens, int wide, int64_t n, const void* w, int64_t vocab, int64_t stride, int d,
                  float scale, void* y, bool vec, int* err, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int64_t items = n * (vec ? d / V : d);
  int64_t blocks = (items + kFwdThreads - 1) / kFwdThreads;
  const int64_t most = static_cast<int64_t>(sm_count()) * 64;
  if (blocks > most) blocks = most;
  if (vec)
    lookup_kernel<T, V><<<static_cast<unsigned>(blocks), kFwdThreads, 0, st>>>(
        tokens, wide, n, static_cast<const T*>(w), vocab, stride, d, scale, static_cast<T*>(y), err);
  else
    lookup_kernel<T, 1><<<static_cast<unsigned>(blocks), kFwdThreads, 0, st>>>(
        tokens, wide, n, static_cast<const T*>(w), vocab, stride, d, scale, static_cast<T*>(y), err);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

constexpr int64_t kMaxTokens = 0x7fffffff;  // positions and keys are 32 bits
constexpr int kMaxWidth = 65536;

int check_sizes(const char* what, int64_t n, int64_t vocab, int d, int token_bits) {
  if (n < 0 || vocab < 1 || d < 1)
    return set_error(OPUS_ERR_INVALID, "%s: bad sizes n=%lld vocab=%lld d=%d", what, (long long)n, (long long)vocab, d);
  if (token_bits != 32 && token_bits != 64)
    return set_error(OPUS_ERR_INVALID, "%s: tokens of %d bits (32 or 64)", what, token_bits);
  if (n > kMaxTokens || vocab > kMaxTokens || d > kMaxWidth)
    return set_error(OPUS_ERR_UNSUPPORTED, "%s: n and vocab up to 2^31 - 1, d up to %d", what, kMaxWidth);
  return OPUS_OK;
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace opus

using namespace opus;

extern "C" int opus_embedding(const void* tokens, int token_bits, int64_t n, const void* weight, int dtype,
                              int64_t vocab, int64_t row_stride, int d, float scale, void* out, void* stream) {
  int rc = check_sizes("embedding", n, vocab, d, token_bits);
  if (rc) return rc;
  if (!dtype_ok(dtype)) return set_error(OPUS_ERR_UNSUPPORTED, "embedding: weight is neither bf16, f16 nor f32");
  if (row_stride < d) return set_error(OPUS_ERR_INVALID, "embedding: row stride %lld < d", (long long)row_stride);
  if (n == 0) return OPUS_OK;
  if (!tokens || !weight || !out) return set_error(OPUS_ERR_INVALID, "embedding: NULL pointer");
  if (!aligned(tokens, token_bits / 8) || !aligned(weight, dtype_bytes(dtype)) || !aligned(out, dtype_bytes(dtype)))
    return set_error(OPUS_ERR_INVALID, "embedding: a pointer is not aligned to its elements");
  int* err = device_error_word();
  if (err == nullptr) return set_error(OPUS_ERR_CUDA, "device error word unavailable");
  const int V = 16 / dtype_bytes(dtype);
  const bool vec = d % V == 0 && row_stride % V == 0 && aligned(weight, 16) && aligned(out, 16);
  const int wide = token_bits == 64;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == OPUS_DTYPE_F32)
    return launch_lookup<float>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
  if (dtype == OPUS_DTYPE_F16)
    return launch_lookup<__half>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
  return launch_lookup<__nv_bfloat16>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
}

extern "C" int64_t opus_embedding_grad_workspace_bytes(int64_t n, int64_t vocab, int d) {
  if (n <= 0 || vocab < 1 || d < 1 || n > kMaxTokens || vocab > kMaxTokens || d > kMaxWidth) return 0;
  return plan_of(n, vocab, d).bytes;
}

extern "C" int opus_embedding_grad(const void* grad_out, int grad_dtype, int64_t row_stride, const void* tokens,
                                   int token_bits, int64_t n, int64_t vocab, int d, float scale, int64_t padding_idx,
                                   void* grad_weight, int out_dtype, int accumulate, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  int rc = check_sizes("embedding_grad", n, vocab, d, token_bits);
  if (rc) return rc;
  if (!dtype_ok(grad_dtype) || (out_dtype != grad_dtype && out_dtype != OPUS_DTYPE_F32))
    return set_error(OPUS_ERR_UNSUPPORTED, "embedding_grad: bf16, f16 or f32 gradients, into their own type or f32");
  if (row_stride < d) return set_error(OPUS_ERR_INVALID, "embedding_grad: row stride %lld < d", (long long)row_stride);
  if (!grad_weight) return set_error(OPUS_ERR_INVALID, "embedding_grad: NULL pointer");
  if (!aligned(grad_weight, dtype_bytes(out_dtype)))
    return set_error(OPUS_ERR_INVALID, "embedding_grad: a pointer is not aligned to its elements");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!accumulate) OPUS_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, vocab * d * dtype_bytes(out_dtype), st));
  if (n == 0) return OPUS_OK;
  if (!grad_out || !tokens || !workspace) return set_error(OPUS_ERR_INVALID, "embedding_grad: NULL pointer");
  if (!aligned(tokens, token_bits / 8) || !aligned(grad_out, dtype_bytes(grad_dtype)))
    return set_error(OPUS_ERR_INVALID, "embedding_grad: a pointer is not aligned to its elements");
  const Plan p = plan_of(n, vocab, d);
  if (workspace_bytes < p.bytes)
    return set_error(OPUS_ERR_INVALID, "embedding_grad: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
                     (long long)p.bytes);
  if (!aligned(workspace, 256)) return set_error(OPUS_ERR_INVALID, "embedding_grad: workspace must be 256-byte aligned");
  int* err = device_error_word();
  if (err == nullptr) return set_error(OPUS_ERR_CUDA, "device error word unavailable");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  KeySource src{tokens, nullptr, nullptr, token_bits == 64, vocab, padding_idx};
  uint32_t *keys = nullptr, *pos = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit;
    const int bits = p.bits - shift < p.digit ? p.bits - shift : p.digit;
    const int tiles = static_cast<int>(p.tiles);
    sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, pass == 0 ? err : nullptr);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    sort_scan_kernel<<<1, kScanThreads, 0, st>>>(counts, p.tiles << bits);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    keys = reinterpret_cast<uint32_t*>(ws + (pass & 1) * 2 * p.keys);
    pos = reinterpret_cast<uint32_t*>(ws + (pass & 1) * 2 * p.keys + p.keys);
    sort_place_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, keys, pos);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    src.keys = keys;
    src.pos = pos;
  }
  const bool f32_out = out_dtype == OPUS_DTYPE_F32;
  const int V = 16 / (f32_out ? 4 : dtype_bytes(grad_dtype));
  const bool vec = d % V == 0 && row_stride % V == 0 && aligned(grad_out, V * dtype_bytes(grad_dtype)) &&
                   aligned(grad_weight, V * dtype_bytes(out_dtype));
  if (grad_dtype == OPUS_DTYPE_F32)
    return launch_sums_by_width<float, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale, accumulate,
                                              grad_weight, parts, st);
  if (grad_dtype == OPUS_DTYPE_F16) {
    if (f32_out)
      return launch_sums_by_width<__half, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                 accumulate, grad_weight, parts, st);
    return launch_sums_by_width<__half, __half>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                accumulate, grad_weight, parts, st);
  }
  if (f32_out)
    return launch_sums_by_width<__nv_bfloat16, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                      accumulate, grad_weight, parts, st);
  return launch_sums_by_width<__nv_bfloat16, __nv_bfloat16>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                            accumulate, grad_weight, parts, st);
}
