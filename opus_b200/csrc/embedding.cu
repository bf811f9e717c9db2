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
// in a workspace, and a second kernel joins them in order.  No sum is made by
// atomics: each has one order, and the result is the same for every call.
// Rows of dW that no token names are zeroed by the same launch as the sums.
//
// Up to 188416 positions are sorted by one cluster of up to 16 blocks that
// hold them in shared memory and exchange them through it (one launch);
// longer lists go through global memory with three launches a pass.
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

constexpr int kFwdRows = 4;  // a thread's, at a time: as many loads in flight

// A thread keeps its column; `across` threads hold a row (of blockIdx.y's part), kFwdThreads / across rows a block.
template <typename T, int V>
__global__ void __launch_bounds__(kFwdThreads) lookup_kernel(const void* __restrict__ tokens, int wide, int64_t n,
                                                             const T* __restrict__ w, int64_t vocab, int64_t stride,
                                                             int d, int across, float scale, T* __restrict__ y, int* err) {
  const int col = (blockIdx.y * across + threadIdx.x % across) * V;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / across);
  if (col >= d) return;
  for (int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.x / across) + threadIdx.x / across; first < n;
       first += step * kFwdRows) {
    int64_t t[kFwdRows];
    Vec<T, V> x[kFwdRows];
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) t[k] = first + k * step < n ? load_token(tokens, wide, first + k * step) : -1;
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) {
      if (t[k] >= 0 && t[k] < vocab) x[k] = *reinterpret_cast<const Vec<T, V>*>(w + t[k] * stride + col);
      else x[k].zero();
    }
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) {
      const int64_t row = first + k * step;
      if (row >= n) break;
      if ((t[k] < 0 || t[k] >= vocab) && col == 0) record_device_error(err, kDevBadToken);
      float r[V];
      x[k].get(r);
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] *= scale;
      store_vec<T, V>(y + row * d + col, r);
    }
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
                                                                  uint32_t* __restrict__ pos_out,
                                                                  uint8_t* __restrict__ present) {
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
    if (present != nullptr && key[r] < src.vocab) present[key[r]] = 1;
  }
}

// ------------------------------------------------------------------ sorting in one cluster
// Block r of the cluster holds the places [r M, (r + 1) M) of the list.  A pass counts digits by warp (a warp's
// items are neighbours), turns the counts into places (over the warps of a block, the blocks before this one, and
// the digits before this one), and stores every item into the block that holds its place.
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kMostBlocks = 16;
constexpr int kMostItems = 11776;  // of a block: four arrays of them and the counts fit its shared memory
constexpr int kItemRounds = (kMostItems + kClusterThreads - 1) / kClusterThreads;
constexpr int kBlockItems = 2048;  // of a block, while there are blocks to share them

struct ClusterSort {
  const void* tokens;
  int wide;
  int n, items;  // items: M
  int64_t vocab, padding;
  int passes, digit, bits;
  uint32_t *keys, *pos;  // sorted
  uint8_t* present;      // vocab bytes (NULL: not wanted): 1 where a key is
  uint32_t* counters;    // two, zeroed
  int* err;
};

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__host__ __device__ constexpr int cluster_sort_bytes(int items) {
  return items * 16 + kClusterWarps * kMaxBins * 2 + kMaxBins * 4 * 2 + 256;
}

__global__ void __launch_bounds__(kClusterThreads, 1) cluster_sort_kernel(const __grid_constant__ ClusterSort p) {
  extern __shared__ __align__(16) uint32_t smem[];
  const int blocks = static_cast<int>(gridDim.x), rank = static_cast<int>(cluster_ctarank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* buffers = smem;  // keys and positions, twice
  uint32_t* totals = smem + 4 * p.items;             // [bins] of this block, read by the others
  uint32_t* base = totals + kMaxBins;                // [bins]
  uint32_t* warp_sums = base + kMaxBins;             // [32] and a spare
  uint16_t* counts = reinterpret_cast<uint16_t*>(warp_sums + 64);  // [warps][bins]
  const int first = rank * p.items;
  const int mine = p.n - first < p.items ? (p.n - first > 0 ? p.n - first : 0) : p.items;
  const int warp_items = ((mine + kClusterWarps - 1) / kClusterWarps + 31) / 32 * 32;
  if (rank == 0 && threadIdx.x < 2) p.counters[threadIdx.x] = 0;
  if (p.present != nullptr) {  // whole words first: the array is padded to 16 bytes
    const int64_t words = (p.vocab + 15) / 16;
    for (int64_t i = rank * kClusterThreads + threadIdx.x; i < words; i += blocks * kClusterThreads)
      reinterpret_cast<uint4*>(p.present)[i] = make_uint4(0, 0, 0, 0);
  }
  for (int i = threadIdx.x; i < mine; i += kClusterThreads) {
    const int64_t t = load_token(p.tokens, p.wide, first + i);
    uint32_t key = static_cast<uint32_t>(p.vocab);
    if (t < 0 || t >= p.vocab) record_device_error(p.err, kDevBadToken);
    else if (t != p.padding) key = static_cast<uint32_t>(t);
    buffers[i] = key;
    buffers[p.items + i] = static_cast<uint32_t>(first + i);
  }
  __syncthreads();
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit;
    const int bins = 1 << (p.bits - shift < p.digit ? p.bits - shift : p.digit);
    const uint32_t* keys = buffers + (pass & 1) * 2 * p.items;
    const uint32_t* pos = keys + p.items;
    const int to = ((pass + 1) & 1) * 2 * p.items;
    for (int i = threadIdx.x; i < kClusterWarps * kMaxBins / 2; i += kClusterThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0;
    __syncthreads();
    uint32_t key[kItemRounds], place[kItemRounds];
    uint16_t* count = counts + warp * kMaxBins;
#pragma unroll
    for (int r = 0; r < kItemRounds; ++r) {
      const int i = warp * warp_items + r * 32 + lane;
      if (r * 32 >= warp_items) continue;  // the same for the whole warp
      const bool live = i < mine;
      key[r] = live ? keys[i] : 0u;
      const uint32_t digit = live ? (key[r] >> shift) & (bins - 1) : kMaxBins;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      const int leader = __ffs(same) - 1;
      uint32_t before = 0;
      if (live && lane == leader) {
        before = count[digit];
        count[digit] = static_cast<uint16_t>(before + __popc(same));
      }
      before = __shfl_sync(0xffffffffu, before, leader);
      place[r] = before + __popc(same & ((1u << lane) - 1));
      __syncwarp();
    }
    __syncthreads();
    const int bin = threadIdx.x;
    uint32_t total = 0;
    if (bin < bins) {
#pragma unroll 8
      for (int w = 0; w < kClusterWarps; ++w) {
        const uint32_t c = counts[w * kMaxBins + bin];
        counts[w * kMaxBins + bin] = static_cast<uint16_t>(total);
        total += c;
      }
      totals[bin] = total;
    }
    __syncwarp();
    cluster_sync();
    uint32_t lower = 0, all = 0;
    if (bin < bins) {
      const uint32_t at = smem_u32(totals + bin);
      for (int r = 0; r < blocks; ++r) {
        const uint32_t c = ld_cluster(mapa_shared(at, r));
        all += c;
        lower += r < rank ? c : 0u;
      }
    }
    // digits before this one: bins <= 512, so the first 16 warps hold them
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (bin < bins) {
      uint32_t before = incl - all + lower;
      for (int w = 0; w < warp; ++w) before += warp_sums[w];
      base[bin] = before;
    }
    __syncthreads();
    const bool done = pass + 1 == p.passes;
#pragma unroll
    for (int r = 0; r < kItemRounds; ++r) {
      const int i = warp * warp_items + r * 32 + lane;
      if (r * 32 >= warp_items || i >= mine) continue;
      const uint32_t digit = (key[r] >> shift) & (bins - 1);
      const uint32_t at = base[digit] + count[digit] + place[r];
      if (done) {
        p.keys[at] = key[r];
        p.pos[at] = pos[i];
        if (p.present != nullptr && key[r] < p.vocab) p.present[key[r]] = 1;
      } else {
        const uint32_t block = at / static_cast<uint32_t>(p.items), slot = at - block * p.items;
        const uint32_t there = mapa_shared(smem_u32(buffers + to + slot), block);
        st_cluster(there, key[r]);
        st_cluster(there + 4u * p.items, pos[i]);
      }
    }
    // items are where the next pass reads them; and no block leaves while another reads its totals
    __syncwarp();
    cluster_sync();
  }
}

// ------------------------------------------------------------------ sums
constexpr int kUnit = 32;         // sorted positions of a unit
constexpr int kSumWarps = 8;      // of a block
constexpr int kBatch = 8;         // rows a warp has in flight
constexpr int kLongUnits = 16;    // a run that goes on for more units is joined by a block, others by a warp

// What the sums leave for the join: runs that cross units, by their first unit.
struct Crossing {
  uint32_t* counters;  // short runs, long runs
  uint32_t* lists;     // [units] short, [units] long
};

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
__device__ void sum_unit(int64_t unit, int slab, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                         int64_t n, int64_t units, uint32_t vocab, const T* __restrict__ dy, int64_t stride, int d,
                         float scale, int accumulate, TO* __restrict__ dw, float* __restrict__ parts,
                         const Crossing& crossing) {
  const int lane = threadIdx.x & 31;
  const int64_t first = unit * kUnit;
  const int col = (slab * 32 + lane) * V;
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
  bool crossed = __shfl_sync(0xffffffffu, my_key, 0) == before;
  for (int b = 0; b < len; b += kBatch) {
    Vec<T, V> x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t p = __shfl_sync(0xffffffffu, my_pos, b + i);  // b + kBatch <= 32
      if (live && b + i < len) x[i] = *reinterpret_cast<const Vec<T, V>*>(dy + static_cast<int64_t>(p) * stride + col);
      else x[i].zero();
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int j = b + i;
      if (j >= len) break;
      float r[V];
      x[i].get(r);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += r[k];
      const uint32_t key = __shfl_sync(0xffffffffu, my_key, j);
      const uint32_t following = __shfl_sync(0xffffffffu, my_key, (j + 1) & 31);
      const uint32_t next = j + 1 < kUnit ? following : after;
      if (next == key && j + 1 < kUnit) continue;
      const bool goes_on = next == key;  // behind the unit's end
      if (live) {
        if (crossed) store_vec<float, V>(parts + (unit * 2) * d + col, acc);
        else if (goes_on) store_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
        else write_row<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc, scale, accumulate);
      }
      if (goes_on && !crossed && slab == 0 && lane == 0) {
        const int64_t far = (unit + 1 + kLongUnits) * kUnit;
        const int is_long = far < n && keys[far] == key;
        crossing.lists[is_long * units + atomicAdd(crossing.counters + is_long, 1u)] = static_cast<uint32_t>(unit);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] = 0.f;
      crossed = false;
    }
  }
}

// Blocks below sum_blocks sum units; the others zero the rows that no token names, a warp 32 neighbouring rows.
template <typename T, typename TO, int V>
__global__ void __launch_bounds__(kSumWarps * 32) sum_kernel(const uint32_t* __restrict__ keys,
                                                             const uint32_t* __restrict__ pos, int64_t n,
                                                             uint32_t vocab, const T* __restrict__ dy, int64_t stride,
                                                             int d, float scale, int accumulate,
                                                             TO* __restrict__ dw, float* __restrict__ parts,
                                                             const __grid_constant__ Crossing crossing,
                                                             const uint8_t* __restrict__ present, unsigned sum_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < sum_blocks) {
    const int slabs = (d / V + 31) / 32;
    const int64_t units = (n + kUnit - 1) / kUnit;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kSumWarps + warp;
    if (item >= units * slabs) return;
    sum_unit<T, TO, V>(item / slabs, static_cast<int>(item % slabs), keys, pos, n, units, vocab, dy, stride, d, scale,
                       accumulate, dw, parts, crossing);
    return;
  }
  const int64_t warps = static_cast<int64_t>(gridDim.x - sum_blocks) * kSumWarps;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x - sum_blocks) * kSumWarps + warp) * 32; r < vocab; r += warps * 32) {
    unsigned absent = __ballot_sync(0xffffffffu, r + lane < vocab && present[r + lane] == 0);
    while (absent != 0) {
      const int64_t row = r + __ffs(absent) - 1;
      absent &= absent - 1;
      Vec<TO, V> zero;
      zero.zero();
      for (int col = lane * V; col < d; col += 32 * V) *reinterpret_cast<Vec<TO, V>*>(dw + row * d + col) = zero;
    }
  }
}

// Sums parts[u][0] over the units [a, b) behind a run's first.
template <int V>
__device__ __forceinline__ void sum_parts(const float* __restrict__ parts, int64_t a, int64_t b, int d, int col, float (&acc)[V]) {
#pragma unroll 8
  for (int64_t u = a; u < b; ++u) {
    float x[V];
    load_vec<float, V>(parts + (u * 2) * d + col, x);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += x[k];
  }
}

// Joins the parts of runs that cross units: a long run and slab of columns by a block, in 32 slices of its units
// that meet in order, a short one by a warp.
constexpr int kJoinWarps = 32;
template <typename TO, int V>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const uint32_t* __restrict__ keys, int64_t n, int d,
                                                               float scale, int accumulate, TO* __restrict__ dw,
                                                               const float* __restrict__ parts,
                                                               const __grid_constant__ Crossing crossing) {
  __shared__ float slice[kJoinWarps][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slabs = (d / V + 31) / 32;
  const int64_t units = (n + kUnit - 1) / kUnit;
  const int64_t n_short = static_cast<int64_t>(crossing.counters[0]) * slabs;
  const int64_t n_long = static_cast<int64_t>(crossing.counters[1]) * slabs;
  for (int64_t item = blockIdx.x; item < n_long; item += gridDim.x) {
    const int64_t unit = crossing.lists[units + item / slabs];
    const int col = (static_cast<int>(item % slabs) * 32 + lane) * V;
    const uint32_t key = keys[(unit + 1) * kUnit];
    int64_t more = 0;  // units behind the first that hold parts of the run: a prefix of those that follow
    while (true) {
      const int64_t u = unit + 1 + more + threadIdx.x;
      const int in = __syncthreads_count(u < units && keys[u * kUnit] == key);
      more += in;
      if (in < kJoinWarps * 32) break;
    }
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
    if (col < d) {
      if (warp == 0) load_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
      sum_parts<V>(parts, unit + 1 + more * warp / kJoinWarps, unit + 1 + more * (warp + 1) / kJoinWarps, d, col, acc);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) slice[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    if (warp == 0 && col < d) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        for (int w = 1; w < kJoinWarps; ++w) acc[k] += slice[w][k * 32 + lane];
      }
      write_row<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc, scale, accumulate);
    }
    __syncthreads();
  }
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kJoinWarps + warp; item < n_short;
       item += static_cast<int64_t>(gridDim.x) * kJoinWarps) {
    const int64_t unit = crossing.lists[item / slabs];
    const int col = (static_cast<int>(item % slabs) * 32 + lane) * V;
    const uint32_t key = keys[(unit + 1) * kUnit];
    const int64_t u = unit + 1 + lane;
    const int more = __popc(__ballot_sync(0xffffffffu, u < units && keys[u * kUnit] == key));  // kLongUnits + 1 at most
    if (col >= d) continue;
    float acc[V];
    load_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
    sum_parts<V>(parts, unit + 1, unit + 1 + more, d, col, acc);
    write_row<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc, scale, accumulate);
  }
}
static_assert(kLongUnits + 1 <= 32, "a warp looks at a short run's units at once");

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int bits, passes, digit;
  bool cluster;  // sorted by one cluster
  int64_t tiles, units;
  // offsets: sorted keys and positions; the counters and lists of crossing runs; the rows' flags; the parts; for
  // the sort through global memory its second keys and positions and its counts
  int64_t keys, crossing, present, parts, second, counts, bytes;
};

Plan plan_of(int64_t n, int64_t vocab, int d) {
  Plan p{};
  while ((vocab >> p.bits) != 0) ++p.bits;  // the key V itself is used
  p.passes = (p.bits + kMaxBits - 1) / kMaxBits;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.tiles = (n + kTile - 1) / kTile;
  p.units = (n + kUnit - 1) / kUnit;
  p.cluster = n <= static_cast<int64_t>(kMostBlocks) * kMostItems;
  p.keys = align256(n * 4);
  p.crossing = 2 * p.keys;
  p.present = p.crossing + 256 + align256(p.units * 8);
  p.parts = p.present + align256(vocab);
  p.second = p.parts + align256(p.units * 2 * d * 4);
  p.counts = p.second + (p.cluster ? 0 : 2 * p.keys);
  p.bytes = p.counts + (p.cluster ? 0 : align256((p.tiles << p.digit) * 4));
  return p;
}

template <typename T, typename TO, int V>
int launch_sums(const uint32_t* keys, const uint32_t* pos, const Plan& p, int64_t n, int64_t vocab, const void* dy,
                int64_t stride, int d, float scale, int accumulate, void* dw, uint8_t* ws, cudaStream_t st) {
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws + p.crossing);
  const Crossing crossing{counters, counters + 64};
  const int64_t slabs = (d / V + 31) / 32, items = p.units * slabs;
  const int64_t sum_blocks = (items + kSumWarps - 1) / kSumWarps;
  int64_t zero_blocks = accumulate ? 0 : (vocab + 32 * kSumWarps - 1) / (32 * kSumWarps);
  const int64_t most = static_cast<int64_t>(sm_count()) * 8;
  zero_blocks = zero_blocks < most ? zero_blocks : most;
  if (sum_blocks + zero_blocks > 0x7fffffff) return set_error(OPUS_ERR_UNSUPPORTED, "embedding_grad: too many positions");
  sum_kernel<T, TO, V><<<static_cast<unsigned>(sum_blocks + zero_blocks), kSumWarps * 32, 0, st>>>(
      keys, pos, n, static_cast<uint32_t>(vocab), static_cast<const T*>(dy), stride, d, scale, accumulate,
      static_cast<TO*>(dw), parts, crossing, ws + p.present, static_cast<unsigned>(sum_blocks));
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  if (p.units < 2) return OPUS_OK;  // nothing crosses
  const int64_t want = (items + kJoinWarps - 1) / kJoinWarps;
  join_kernel<TO, V><<<static_cast<unsigned>(want < 2 * sm_count() ? want : 2 * sm_count()), kJoinWarps * 32, 0, st>>>(
      keys, n, d, scale, accumulate, static_cast<TO*>(dw), parts, crossing);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename T, typename TO>
int launch_sums_by_width(bool wide, const uint32_t* keys, const uint32_t* pos, const Plan& p, int64_t n, int64_t vocab,
                         const void* dy, int64_t stride, int d, float scale, int accumulate, void* dw, uint8_t* ws,
                         cudaStream_t st) {
  constexpr int V = 16 / (sizeof(T) > sizeof(TO) ? sizeof(T) : sizeof(TO));
  if (wide) return launch_sums<T, TO, V>(keys, pos, p, n, vocab, dy, stride, d, scale, accumulate, dw, ws, st);
  return launch_sums<T, TO, 1>(keys, pos, p, n, vocab, dy, stride, d, scale, accumulate, dw, ws, st);
}

int launch_cluster_sort(const Plan& p, const KeySource& src, int64_t n, uint8_t* ws, bool flags, int* err, cudaStream_t st) {
  int blocks = 1;
  while (blocks < kMostBlocks && static_cast<int64_t>(blocks) * kBlockItems < n) blocks *= 2;
  ClusterSort a{};
  a.tokens = src.tokens, a.wide = src.wide, a.vocab = src.vocab, a.padding = src.padding;
  a.n = static_cast<int>(n);
  a.items = static_cast<int>(((n + blocks - 1) / blocks + 31) / 32 * 32);
  a.passes = p.passes, a.digit = p.digit, a.bits = p.bits;
  a.keys = reinterpret_cast<uint32_t*>(ws);
  a.pos = reinterpret_cast<uint32_t*>(ws + p.keys);
  a.present = flags ? ws + p.present : nullptr;
  a.counters = reinterpret_cast<uint32_t*>(ws + p.crossing);
  a.err = err;
  const int shared = cluster_sort_bytes(a.items);
  OPUS_CUDA_TRY(cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
  OPUS_CUDA_TRY(cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks), cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = shared, cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
  OPUS_CUDA_TRY(cudaLaunchKernelEx(&cfg, cluster_sort_kernel, a));
  note_launch();
  return OPUS_OK;
}

int launch_global_sort(const Plan& p, KeySource src, int64_t n, uint8_t* ws, bool flags, int* err, cudaStream_t st) {
  OPUS_CUDA_TRY(cudaMemsetAsync(ws + p.crossing, 0, 8, st));
  if (flags) OPUS_CUDA_TRY(cudaMemsetAsync(ws + p.present, 0, src.vocab, st));
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  const int tiles = static_cast<int>(p.tiles);
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit;
    const int bits = p.bits - shift < p.digit ? p.bits - shift : p.digit;
    const bool last = pass + 1 == p.passes;
    sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, pass == 0 ? err : nullptr);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    sort_scan_kernel<<<1, kScanThreads, 0, st>>>(counts, p.tiles << bits);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    // the last pass ends in the first pair of arrays
    uint8_t* to = ws + ((p.passes - pass) % 2 == 1 ? 0 : p.second);
    uint32_t* keys = reinterpret_cast<uint32_t*>(to);
    uint32_t* pos = reinterpret_cast<uint32_t*>(to + p.keys);
    sort_place_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, keys, pos,
                                                      last && flags ? ws + p.present : nullptr);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    src.keys = keys;
    src.pos = pos;
  }
  return OPUS_OK;
}

template <typename T>
int launch_lookup(const void* tokens, int wide, int64_t n, const void* w, int64_t vocab, int64_t stride, int d,
                  float scale, void* y, bool vec, int* err, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int per_row = vec ? d / V : d;
  const int parts = (per_row + kFwdThreads - 1) / kFwdThreads, across = (per_row + parts - 1) / parts;
  const int rows = kFwdThreads / across;  // of a block
  int64_t blocks = (n + rows * kFwdRows - 1) / (rows * kFwdRows);
  const int64_t most = static_cast<int64_t>(sm_count()) * 64;
  if (blocks > most) blocks = most;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(parts));
  if (vec)
    lookup_kernel<T, V><<<grid, rows * across, 0, st>>>(tokens, wide, n, static_cast<const T*>(w), vocab, stride, d,
                                                        across, scale, static_cast<T*>(y), err);
  else
    lookup_kernel<T, 1><<<grid, rows * across, 0, st>>>(tokens, wide, n, static_cast<const T*>(w), vocab, stride, d,
                                                        across, scale, static_cast<T*>(y), err);
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
  if (n == 0) {
    if (!accumulate) OPUS_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, vocab * d * dtype_bytes(out_dtype), st));
    return OPUS_OK;
  }
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
  const KeySource src{tokens, nullptr, nullptr, token_bits == 64, vocab, padding_idx};
  rc = p.cluster ? launch_cluster_sort(p, src, n, ws, !accumulate, err, st)
                 : launch_global_sort(p, src, n, ws, !accumulate, err, st);
  if (rc) return rc;
  const uint32_t* keys = reinterpret_cast<const uint32_t*>(ws);
  const uint32_t* pos = reinterpret_cast<const uint32_t*>(ws + p.keys);
  const bool f32_out = out_dtype == OPUS_DTYPE_F32;
  const int V = 16 / (f32_out ? 4 : dtype_bytes(grad_dtype));
  const bool vec = d % V == 0 && row_stride % V == 0 && aligned(grad_out, V * dtype_bytes(grad_dtype)) &&
                   aligned(grad_weight, V * dtype_bytes(out_dtype));
  if (grad_dtype == OPUS_DTYPE_F32)
    return launch_sums_by_width<float, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale, accumulate,
                                              grad_weight, ws, st);
  if (grad_dtype == OPUS_DTYPE_F16) {
    if (f32_out)
      return launch_sums_by_width<__half, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                 accumulate, grad_weight, ws, st);
    return launch_sums_by_width<__half, __half>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                accumulate, grad_weight, ws, st);
  }
  if (f32_out)
    return launch_sums_by_width<__nv_bfloat16, float>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                      accumulate, grad_weight, ws, st);
  return launch_sums_by_width<__nv_bfloat16, __nv_bfloat16>(vec, keys, pos, p, n, vocab, grad_out, row_stride, d, scale,
                                                            accumulate, grad_weight, ws, st);
}
