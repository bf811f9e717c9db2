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
//
// Up to 188416 positions are sorted by one cluster of up to 16 blocks that
// hold them in shared memory and exchange them through it (one launch), while
// the other multiprocessors zero dW; longer lists go through global memory
// with three launches a pass.
//
// Tokens outside [0, V) give a row of zeros, add to no gradient, and are
// recorded in the device's error word for tokens.  Tokens equal to padding_idx add to no
// gradient.
//
// Bound: HBM bandwidth.  The lookup is a stream of writes: 147456 rows of 1600
// bf16 elements in 95 to 97 us, 4.9 TB/s written (a memset on the same
// device writes 3.9, a copy moves 6.5).  The gradient reads dY once, whole rows in sorted
// order, and writes dW, the named rows twice (zeros, then sums: the zeroing
// hides behind the sort, which leaves HBM idle): 81920 x 768 f32 tokens of a
// 50257-row table in 102 us (a profile gives 35 to sort and zero, 50 to sum and
// 16 to join); 16384 x 2048 bf16 of a 151936-row table in 121 to 137 us, where a
// memset of dW alone takes 160.  Lists between those and the short ones (below)
// are bound by the chain of three launches: 19 to 25 us.
#include <algorithm>

#include "elements.cuh"
#include "per_device.h"

namespace opus {
namespace {

constexpr int kFwdThreads = 256;
constexpr int kFwdBlocksPerSm = 6;

__device__ __forceinline__ int64_t load_token(const void* tokens, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(tokens)[i] : static_cast<const int32_t*>(tokens)[i];
}

constexpr int kFwdRows = 4;  // a thread's, at a time: as many loads in flight

// A thread keeps its column; `across` threads hold a row (of blockIdx.y's part), blockDim.x / across rows a block.
// Scaled: with a scale other than 1, which leaves rows as they are.
template <typename T, int V, typename Token, bool Scaled>
__global__ void __launch_bounds__(kFwdThreads) lookup_kernel(const Token* __restrict__ tokens, int64_t n,
                                                             const T* __restrict__ w, int64_t vocab, int64_t stride,
                                                             int d, int across, float scale, T* __restrict__ y, int* err) {
  const int col = (blockIdx.y * across + threadIdx.x % across) * V;
  if (col >= d) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / across);
  int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.x / across) + threadIdx.x / across;
  const T* from = w + col;
  T* to = y + first * d + col;
  const int64_t to_step = step * d;
  for (; first < n; first += step * kFwdRows) {
    int64_t t[kFwdRows];
    Vec<T, V> x[kFwdRows];
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) {
      t[k] = first + k * step < n ? static_cast<int64_t>(tokens[first + k * step]) : -1;
    }
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) {
      if (static_cast<uint64_t>(t[k]) < static_cast<uint64_t>(vocab)) {
        x[k] = *reinterpret_cast<const Vec<T, V>*>(from + t[k] * stride);
      } else {
        x[k].zero();
        if (col == 0 && first + k * step < n) record_device_error(err, kDevBadToken);
      }
    }
#pragma unroll
    for (int k = 0; k < kFwdRows; ++k) {
      if (first + k * step < n) {
        if constexpr (Scaled) {
          float r[V];
          x[k].get(r);
#pragma unroll
          for (int i = 0; i < V; ++i) r[i] *= scale;
          x[k].set(r);
        }
        *reinterpret_cast<Vec<T, V>*>(to) = x[k];
      }
      to += to_step;
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
  const void* tokens;  // first pass; later passes read items (key, position)
  const uint2* items;
  int wide;
  int64_t vocab;
  int64_t padding;
};

__device__ __forceinline__ uint2 load_item(const KeySource& s, int64_t i, int* err) {
  if (s.items != nullptr) return s.items[i];
  uint2 item = make_uint2(static_cast<uint32_t>(s.vocab), static_cast<uint32_t>(i));
  const int64_t t = load_token(s.tokens, s.wide, i);
  if (t < 0 || t >= s.vocab) {
    record_device_error(err, kDevBadToken);
  } else if (t != s.padding) {
    item.x = static_cast<uint32_t>(t);
  }
  return item;
}

// The lanes whose digit is this lane's, among those in `live`, by a ballot for each bit.
__device__ __forceinline__ unsigned same_digit(uint32_t digit, int bits, unsigned live) {
  unsigned same = live;
#pragma unroll
  for (int b = 0; b < kMaxBits; ++b) {
    if (b >= bits) break;
    const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
    same &= (digit >> b) & 1u ? set : ~set;
  }
  return same;
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
    if (i < n) atomicAdd(&hist[(load_item(src, i, err).x >> shift) & (bins - 1)], 1u);
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
                                                                  uint2* __restrict__ out) {
  __shared__ uint32_t count[kSortWarps][kMaxBins];
  const int bins = 1 << bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
  __syncthreads();
  // a warp's keys are kSortRounds runs of 32 neighbours: rounds in order keep equal keys in order
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile + warp * (32 * kSortRounds) + lane;
  uint2 item[kSortRounds];
  uint32_t place[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * 32;
    const bool live = i < n;
    item[r] = live ? load_item(src, i, nullptr) : make_uint2(0u, 0u);
    const uint32_t digit = (item[r].x >> shift) & (bins - 1);
    const unsigned same = same_digit(digit, bits, __ballot_sync(0xffffffffu, live)) | (live ? 0u : 1u << lane);
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
    out[count[warp][(item[r].x >> shift) & (bins - 1)] + place[r]] = item[r];
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
constexpr int kBlockItems = 2048;  // of a block, while there are blocks to share them: 10 to 12 us for one block
                                   // (zeros of a 51 MB table with it), 14 for 16384 on eight, 24 for 81920 and 36 for
                                   // 147456 on sixteen

struct ClusterSort {
  const void* tokens;
  int wide;
  int n, items;  // items: M
  int64_t vocab, padding;
  int passes, digit, bits;
  uint2* sorted;       // (key, position)
  uint32_t* counters;  // two, zeroed
  int blocks;          // of the cluster: cluster 0 sorts, the others zero
  uint8_t* zero;       // zero_bytes from an address that is a multiple of 16, less than 16 more behind them
  int64_t zero_bytes;
  int* err;
};

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}

__host__ __device__ constexpr int cluster_sort_bytes(int items) {
  return items * 16 + kClusterWarps * kMaxBins * 2 + kMaxBins * 4 * 2 + 256;
}

__global__ void __launch_bounds__(kClusterThreads, 1) cluster_sort_kernel(const __grid_constant__ ClusterSort p) {
  extern __shared__ __align__(16) uint32_t smem[];
  const int blocks = p.blocks;
  if (blockIdx.x >= blocks) {  // none of these blocks' clusters sorts
    const int64_t whole = p.zero_bytes / 16, step = static_cast<int64_t>(gridDim.x - blocks) * kClusterThreads;
    int64_t i = (blockIdx.x - blocks) * static_cast<int64_t>(kClusterThreads) + threadIdx.x;
    if (i < p.zero_bytes - whole * 16) p.zero[whole * 16 + i] = 0;
    for (; i < whole; i += step) reinterpret_cast<uint4*>(p.zero)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int rank = static_cast<int>(cluster_ctarank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint2* buffers = reinterpret_cast<uint2*>(smem);   // items, twice
  uint32_t* totals = smem + 4 * p.items;             // [bins] of this block, read by the others
  uint32_t* base = totals + kMaxBins;                // [bins]
  uint32_t* warp_sums = base + kMaxBins;             // [32] and a spare
  uint16_t* counts = reinterpret_cast<uint16_t*>(warp_sums + 64);  // [warps][bins]
  const int first = rank * p.items;
  const int mine = p.n - first < p.items ? (p.n - first > 0 ? p.n - first : 0) : p.items;
  const int warp_items = ((mine + kClusterWarps - 1) / kClusterWarps + 31) / 32 * 32;
  if (rank == 0 && threadIdx.x < 2) p.counters[threadIdx.x] = 0;
  const KeySource src{p.tokens, nullptr, p.wide, p.vocab, p.padding};
#pragma unroll 4
  for (int i = threadIdx.x; i < mine; i += kClusterThreads) buffers[i] = load_item(src, first + i, p.err);
  __syncthreads();
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit;
    const int bits = p.bits - shift < p.digit ? p.bits - shift : p.digit, bins = 1 << bits;
    const uint2* items = buffers + (pass & 1) * p.items;
    uint2* to = buffers + ((pass + 1) & 1) * p.items;
    for (int i = threadIdx.x; i < kClusterWarps * kMaxBins / 2; i += kClusterThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0;
    __syncthreads();
    uint2 item[kItemRounds];
    uint32_t place[kItemRounds];
    uint16_t* count = counts + warp * kMaxBins;
#pragma unroll
    for (int r = 0; r < kItemRounds; ++r) {
      const int i = warp * warp_items + r * 32 + lane;
      if (r * 32 >= warp_items) continue;  // the same for the whole warp
      const bool live = i < mine;
      item[r] = live ? items[i] : make_uint2(0u, 0u);
      const uint32_t digit = (item[r].x >> shift) & (bins - 1);
      const unsigned same = same_digit(digit, bits, __ballot_sync(0xffffffffu, live)) | (live ? 0u : 1u << lane);
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
      uint32_t c[kClusterWarps];  // all loads first: they wait together
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) c[w] = counts[w * kMaxBins + bin];
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) {
        counts[w * kMaxBins + bin] = static_cast<uint16_t>(total);
        total += c[w];
      }
      totals[bin] = total;
    }
    __syncwarp();
    cluster_sync();
    uint32_t lower = 0, all = 0;
    if (bin < bins) {
      const uint32_t at = smem_u32(totals + bin);
      uint32_t c[kMostBlocks];
#pragma unroll
      for (int r = 0; r < kMostBlocks; ++r) c[r] = r < blocks ? ld_cluster(mapa_shared(at, r)) : 0u;
#pragma unroll
      for (int r = 0; r < kMostBlocks; ++r) {
        all += c[r];
        lower += r < rank ? c[r] : 0u;
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
    uint32_t before = lane < warp ? warp_sums[lane] : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (bin < bins) base[bin] = before + incl - all + lower;
    __syncthreads();
    const bool done = pass + 1 == p.passes;
#pragma unroll
    for (int r = 0; r < kItemRounds; ++r) {
      const int i = warp * warp_items + r * 32 + lane;
      if (r * 32 >= warp_items || i >= mine) continue;
      const uint32_t digit = (item[r].x >> shift) & (bins - 1);
      const uint32_t at = base[digit] + count[digit] + place[r];
      if (done) {
        p.sorted[at] = item[r];
      } else {
        const uint32_t block = at / static_cast<uint32_t>(p.items), slot = at - block * p.items;
        st_cluster(mapa_shared(smem_u32(to + slot), block), item[r]);
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
constexpr int kLongUnits = 31;    // a run that goes on for more units is joined by a block, others by a warp

// What the sums leave for the join: runs that cross units, by their first unit.
struct Crossing {
  uint32_t* counters;  // short runs, long runs
  uint2* lists;        // [units] short, [units] long: unit, key
};

template <typename TO, int V, bool Add>
__device__ __forceinline__ void write_row(TO* out, const float (&acc)[V], float scale) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = acc[k] * scale;
  if constexpr (Add) {
    float o[V];
    load_vec<TO, V>(out, o);
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] += o[k];
  }
  store_vec<TO, V>(out, r);
}

// One warp: one unit, 32 * V columns.  parts[unit]: [0] the part of a run that came from the unit before (or
// fills the unit), [1] the part of a run that starts here and goes on.  Add: into what is there (a batch's rows of
// dW are loaded with its rows of dY: loaded where a run ends, each would be waited for on its own).
template <typename T, typename TO, int V, bool Add>
__device__ void sum_unit(int64_t unit, int slab, const uint2* __restrict__ sorted, int64_t n, int64_t units,
                         uint32_t vocab, const T* __restrict__ dy, int64_t stride, int d, float scale,
                         TO* __restrict__ dw, float* __restrict__ parts, const Crossing& crossing) {
  constexpr int kBatch = Add ? 4 : 8;  // rows in flight (with rows of dW, 8 took registers for two blocks of five)
  const int lane = threadIdx.x & 31;
  const int64_t first = unit * kUnit;
  const int col = (slab * 32 + lane) * V;
  const bool live = col < d;
  const int64_t mine = first + lane;
  const uint2 item = mine < n ? sorted[mine] : make_uint2(vocab, 0u);
  const uint32_t my_key = item.x, my_pos = item.y;
  const uint32_t before = first > 0 ? sorted[first - 1].x : vocab;
  const uint32_t after = first + kUnit < n ? sorted[first + kUnit].x : vocab;
  const int len = __popc(__ballot_sync(0xffffffffu, my_key < vocab));  // keys equal to vocab sort last
  const uint32_t my_next = __shfl_down_sync(0xffffffffu, my_key, 1);
  const unsigned ends = __ballot_sync(0xffffffffu, lane == 31 || my_next != my_key);  // runs end, or the unit does
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.f;
  bool crossed = __shfl_sync(0xffffffffu, my_key, 0) == before;
  for (int b = 0; b < len; b += kBatch) {
    Vec<T, V> x[kBatch];
    Vec<TO, V> o[Add ? kBatch : 1];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t p = __shfl_sync(0xffffffffu, my_pos, b + i);  // b + kBatch <= 32
      if (live && b + i < len) x[i] = *reinterpret_cast<const Vec<T, V>*>(dy + static_cast<int64_t>(p) * stride + col);
      else x[i].zero();
    }
    if constexpr (Add) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t key = __shfl_sync(0xffffffffu, my_key, b + i);
        if (live && b + i < len && (ends >> (b + i) & 1u)) o[i] = *reinterpret_cast<const Vec<TO, V>*>(dw + static_cast<int64_t>(key) * d + col);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int j = b + i;
      if (j >= len) break;
      float r[V];
      x[i].get(r);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += r[k];
      if ((ends >> j & 1u) == 0) continue;
      const uint32_t key = __shfl_sync(0xffffffffu, my_key, j);
      const bool goes_on = j + 1 == kUnit && after == key;
      if (live) {
        if (crossed) {
          store_vec<float, V>(parts + (unit * 2) * d + col, acc);
        } else if (goes_on) {
          store_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
        } else {
          if constexpr (Add) {
            float old[V];
            o[i].get(old);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = acc[k] * scale + old[k];
          } else {
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] *= scale;
          }
          store_vec<TO, V>(dw + static_cast<int64_t>(key) * d + col, acc);
        }
      }
      if (goes_on && !crossed && slab == 0 && lane == 0) {
        const int64_t far = (unit + 1 + kLongUnits) * kUnit;
        const int is_long = far < n && sorted[far].x == key;
        crossing.lists[is_long * units + atomicAdd(crossing.counters + is_long, 1u)] = make_uint2(static_cast<uint32_t>(unit), key);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] = 0.f;
      crossed = false;
    }
  }
}

template <typename T, typename TO, int V, bool Add>
__global__ void __launch_bounds__(kSumWarps * 32) sum_kernel(const uint2* __restrict__ sorted, int64_t n, uint32_t vocab,
                                                             const T* __restrict__ dy, int64_t stride, int d, float scale,
                                                             TO* __restrict__ dw, float* __restrict__ parts,
                                                             const __grid_constant__ Crossing crossing) {
  wait_for_predecessors();
  const int slabs = (d / V + 31) / 32;
  const int64_t units = (n + kUnit - 1) / kUnit;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
  if (item < units * slabs)
    sum_unit<T, TO, V, Add>(item / slabs, static_cast<int>(item % slabs), sorted, n, units, vocab, dy, stride, d, scale,
                            dw, parts, crossing);
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

// Joins the parts of runs that cross units: a long run and slab of columns by a block (from the grid's first), in
// 32 slices of its units that meet in order, a short one by a warp (from the grid's last).
constexpr int kJoinWarps = 32;
template <typename TO, int V, bool Add>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const uint2* __restrict__ sorted, int64_t n, int d,
                                                               float scale, TO* __restrict__ dw,
                                                               const float* __restrict__ parts,
                                                               const __grid_constant__ Crossing crossing) {
  __shared__ float slice[kJoinWarps][32 * V];
  wait_for_predecessors();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slabs = (d / V + 31) / 32;
  const int64_t units = (n + kUnit - 1) / kUnit;
  const int64_t n_short = static_cast<int64_t>(crossing.counters[0]) * slabs;
  const int64_t n_long = static_cast<int64_t>(crossing.counters[1]) * slabs;
  for (int64_t item = blockIdx.x; item < n_long; item += gridDim.x) {
    const uint2 run = crossing.lists[units + item / slabs];
    const int64_t unit = run.x;
    const int col = (static_cast<int>(item % slabs) * 32 + lane) * V;
    int64_t more = 0;  // units behind the first that hold parts of the run: a prefix of those that follow
    while (true) {
      const int64_t u = unit + 1 + more + threadIdx.x;
      const int in = __syncthreads_count(u < units && sorted[u * kUnit].x == run.y);
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
    // slices w and w + half, until one is left
#pragma unroll
    for (int half = kJoinWarps / 2; half > 0; half >>= 1) {
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int k = 0; k < V; ++k) slice[warp][k * 32 + lane] = acc[k];
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += slice[warp + half][k * 32 + lane];
      }
    }
    if (warp == 0 && col < d) write_row<TO, V, Add>(dw + static_cast<int64_t>(run.y) * d + col, acc, scale);
    __syncthreads();
  }
  for (int64_t item = static_cast<int64_t>(gridDim.x - 1 - blockIdx.x) * kJoinWarps + warp; item < n_short;
       item += static_cast<int64_t>(gridDim.x) * kJoinWarps) {
    const uint2 run = crossing.lists[item / slabs];
    const int64_t unit = run.x, u = unit + 1 + lane;
    const int col = (static_cast<int>(item % slabs) * 32 + lane) * V;
    const int more = __popc(__ballot_sync(0xffffffffu, u < units && sorted[u * kUnit].x == run.y));  // kLongUnits at most
    if (col >= d) continue;
    float acc[V];
    load_vec<float, V>(parts + (unit * 2 + 1) * d + col, acc);
    sum_parts<V>(parts, unit + 1, unit + 1 + more, d, col, acc);
    write_row<TO, V, Add>(dw + static_cast<int64_t>(run.y) * d + col, acc, scale);
  }
}
static_assert(kLongUnits < 32, "a warp looks at a short run's units at once");

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int bits, passes, digit;
  bool cluster;  // sorted by one cluster
  int64_t tiles, units;
  // offsets: the sorted items; the counters and lists of crossing runs; the parts; for the sort through global
  // memory its second items and its counts
  int64_t crossing, parts, second, counts, bytes;
};

Plan plan_of(int64_t n, int64_t vocab, int d) {
  Plan p{};
  while ((vocab >> p.bits) != 0) ++p.bits;  // the key V itself is used
  p.passes = (p.bits + kMaxBits - 1) / kMaxBits;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.tiles = (n + kTile - 1) / kTile;
  p.units = (n + kUnit - 1) / kUnit;
  p.cluster = n <= static_cast<int64_t>(kMostBlocks) * kMostItems;
  p.crossing = align256(n * 8);
  p.parts = p.crossing + 256 + align256(p.units * 16);
  p.second = p.parts + align256(p.units * 2 * d * 4);
  p.counts = p.second + (p.cluster ? 0 : align256(n * 8));
  p.bytes = p.counts + (p.cluster ? 0 : align256((p.tiles << p.digit) * 4));
  return p;
}

template <typename T, typename TO, int V, bool Add>
int launch_sums(const Plan& p, int64_t n, int64_t vocab, const void* dy, int64_t stride, int d, float scale, void* dw,
                uint8_t* ws, cudaStream_t st) {
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws + p.crossing);
  const Crossing crossing{counters, reinterpret_cast<uint2*>(ws + p.crossing + 256)};
  const int64_t slabs = (d / V + 31) / 32, items = p.units * slabs;
  const int64_t blocks = (items + kSumWarps - 1) / kSumWarps;
  if (blocks > 0x7fffffff) return set_error(OPUS_ERR_UNSUPPORTED, "embedding_grad: too many positions");
  const uint2* sorted = reinterpret_cast<const uint2*>(ws);
  OPUS_CUDA_TRY(launch_early(sum_kernel<T, TO, V, Add>, dim3(static_cast<unsigned>(blocks)), kSumWarps * 32, 0, st, sorted,
                             n, static_cast<uint32_t>(vocab), static_cast<const T*>(dy), stride, d, scale,
                             static_cast<TO*>(dw), parts, crossing));
  note_launch();
  if (p.units < 2) return OPUS_OK;  // nothing crosses
  const int64_t want = (items + kJoinWarps - 1) / kJoinWarps, most = 2 * sm_count();
  OPUS_CUDA_TRY(launch_early(join_kernel<TO, V, Add>, dim3(static_cast<unsigned>(want < most ? want : most)),
                             kJoinWarps * 32, 0, st, sorted, n, d, scale, static_cast<TO*>(dw), parts, crossing));
  note_launch();
  return OPUS_OK;
}

template <typename T, typename TO>
int launch_sums_by_width(bool wide, const Plan& p, int64_t n, int64_t vocab,
                         const void* dy, int64_t stride, int d, float scale, int accumulate, void* dw, uint8_t* ws,
                         cudaStream_t st) {
  constexpr int V = 16 / (sizeof(T) > sizeof(TO) ? sizeof(T) : sizeof(TO));
  if (wide)
    return accumulate ? launch_sums<T, TO, V, true>(p, n, vocab, dy, stride, d, scale, dw, ws, st)
                      : launch_sums<T, TO, V, false>(p, n, vocab, dy, stride, d, scale, dw, ws, st);
  return accumulate ? launch_sums<T, TO, 1, true>(p, n, vocab, dy, stride, d, scale, dw, ws, st)
                    : launch_sums<T, TO, 1, false>(p, n, vocab, dy, stride, d, scale, dw, ws, st);
}

// Clusters of 2^k sorting blocks that the device holds at once (a cluster lies in one group of its
// multiprocessors): one that had to wait for others would begin to zero when they have ended.
int resident_clusters(const cudaLaunchConfig_t& cfg, int k) {
  static PerDevice<5> known;
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess) device = -1;
  return known.get(device, k, 1, [&cfg] {
    int n = 0;
    return cudaOccupancyMaxActiveClusters(&n, cluster_sort_kernel, &cfg) == cudaSuccess ? n : 0;
  });
}

// zero_bytes of zero (0: none) are zeroed by the blocks that do not sort.
int launch_cluster_sort(const Plan& p, const KeySource& src, int64_t n, uint8_t* ws, void* zero, int64_t zero_bytes,
                        int* err, cudaStream_t st) {
  int blocks = 1, k = 0;
  for (; blocks < kMostBlocks && static_cast<int64_t>(blocks) * kBlockItems < n; ++k) blocks *= 2;
  ClusterSort a{};
  a.tokens = src.tokens, a.wide = src.wide, a.vocab = src.vocab, a.padding = src.padding;
  a.n = static_cast<int>(n);
  a.items = static_cast<int>(((n + blocks - 1) / blocks + 31) / 32 * 32);
  a.passes = p.passes, a.digit = p.digit, a.bits = p.bits;
  a.sorted = reinterpret_cast<uint2*>(ws);
  a.counters = reinterpret_cast<uint32_t*>(ws + p.crossing);
  a.blocks = blocks;
  a.err = err;
  // bytes before the first 16-byte boundary are left to a memset of their own
  const int64_t head = zero_bytes > 0 ? (16 - reinterpret_cast<uintptr_t>(zero) % 16) % 16 : 0;
  if (head > 0) OPUS_CUDA_TRY(cudaMemsetAsync(zero, 0, head < zero_bytes ? head : zero_bytes, st));
  a.zero = static_cast<uint8_t*>(zero) + head;
  a.zero_bytes = zero_bytes > head ? zero_bytes - head : 0;
  // every launch takes the shared memory of the longest list: one block a multiprocessor, whatever n
  const int shared = cluster_sort_bytes(kMostItems);
  OPUS_CUDA_TRY(cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
  OPUS_CUDA_TRY(cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks), cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = shared, cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
  int64_t zeroing = (a.zero_bytes + kClusterThreads * 16 * 8 - 1) / (kClusterThreads * 16 * 8);
  zeroing = (zeroing + blocks - 1) / blocks;
  if (zeroing > 0) {
    const int held = resident_clusters(cfg, k) - 1;
    zeroing = zeroing < held ? zeroing : held > 0 ? held : 1;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * (1 + zeroing)));
  OPUS_CUDA_TRY(cudaLaunchKernelEx(&cfg, cluster_sort_kernel, a));
  note_launch();
  return OPUS_OK;
}

int launch_global_sort(const Plan& p, KeySource src, int64_t n, uint8_t* ws, void* zero, int64_t zero_bytes, int* err,
                       cudaStream_t st) {
  if (zero_bytes > 0) OPUS_CUDA_TRY(cudaMemsetAsync(zero, 0, zero_bytes, st));
  OPUS_CUDA_TRY(cudaMemsetAsync(ws + p.crossing, 0, 8, st));
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  const int tiles = static_cast<int>(p.tiles);
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit;
    const int bits = p.bits - shift < p.digit ? p.bits - shift : p.digit;
    sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, pass == 0 ? err : nullptr);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    sort_scan_kernel<<<1, kScanThreads, 0, st>>>(counts, p.tiles << bits);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    // the last pass ends in the first array
    uint2* to = reinterpret_cast<uint2*>(ws + ((p.passes - pass) % 2 == 1 ? 0 : p.second));
    sort_place_kernel<<<tiles, kSortThreads, 0, st>>>(src, n, shift, bits, tiles, counts, to);
    note_launch();
    OPUS_CUDA_TRY(cudaGetLastError());
    src.items = to;
  }
  return OPUS_OK;
}

template <typename T, int V, typename Token, bool Scaled>
int launch_lookup(const void* tokens, int64_t n, const void* w, int64_t vocab, int64_t stride, int d, float scale,
                  void* y, int* err, cudaStream_t st) {
  constexpr auto kernel = lookup_kernel<T, V, Token, Scaled>;
  const int per_row = d / V;
  const int parts = (per_row + kFwdThreads - 1) / kFwdThreads, across = (per_row + parts - 1) / parts;
  const int rows = kFwdThreads / across;  // of a block
  // blocks that stay: what a thread sets up serves many rows
  const int64_t need = (n + rows * kFwdRows - 1) / (rows * kFwdRows);
  const int64_t most = (static_cast<int64_t>(sm_count()) * kFwdBlocksPerSm + parts - 1) / parts;
  const dim3 grid(static_cast<unsigned>(need < most ? need : most), static_cast<unsigned>(parts));
  kernel<<<grid, rows * across, 0, st>>>(static_cast<const Token*>(tokens), n, static_cast<const T*>(w), vocab, stride, d,
                                         across, scale, static_cast<T*>(y), err);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename T, int V>
int launch_lookup_by_token(const void* tokens, int wide, int64_t n, const void* w, int64_t vocab, int64_t stride, int d,
                           float scale, void* y, int* err, cudaStream_t st) {
  if (wide)
    return scale == 1.0f ? launch_lookup<T, V, int64_t, false>(tokens, n, w, vocab, stride, d, scale, y, err, st)
                         : launch_lookup<T, V, int64_t, true>(tokens, n, w, vocab, stride, d, scale, y, err, st);
  return scale == 1.0f ? launch_lookup<T, V, int32_t, false>(tokens, n, w, vocab, stride, d, scale, y, err, st)
                       : launch_lookup<T, V, int32_t, true>(tokens, n, w, vocab, stride, d, scale, y, err, st);
}

template <typename T>
int launch_lookup_by_width(const void* tokens, int wide, int64_t n, const void* w, int64_t vocab, int64_t stride, int d,
                           float scale, void* y, bool vec, int* err, cudaStream_t st) {
  return vec ? launch_lookup_by_token<T, 16 / sizeof(T)>(tokens, wide, n, w, vocab, stride, d, scale, y, err, st)
             : launch_lookup_by_token<T, 1>(tokens, wide, n, w, vocab, stride, d, scale, y, err, st);
}

// ---- short lists: one launch
// Every block holds the whole list.  It zeroes its share of the rows that no token names, and sums the tokens that
// occur first at its positions.  A token's few occurrences are summed by every warp for columns of its own; many are
// cut among the warps, whose sums are joined in order.  No row is written twice.
//
// One launch instead of three: 300 tokens of 80 f32 columns 6 us instead of 19, 300 of 768 bf16 18 instead of 24 (a
// table of 77 MB to zero).  What it does badly is a token that fills the list: 0.44 us for each 64 positions and each
// 32 vectors of columns (2048 positions of 1600 f32 columns, two tokens: 185 us, 16 sorted), so lists are short while
// that product is 32 at most (14 us, 19 sorted, at 2048 x 80).
constexpr int kShortList = 2048;
constexpr int64_t kShortWork = 32;
constexpr int kShortThreads = 256, kShortWarps = kShortThreads / 32;
constexpr int kShortFlags = 1024;    // words: a bit for each row of a block's share
constexpr int kShortBlocksPerSm = 4;
constexpr int kShortSerial = 32;     // occurrences that each warp sums alone

template <typename T, int V>
__device__ __forceinline__ void add_rows(const uint32_t* at, int count, const T* __restrict__ dy, int64_t stride,
                                         float (&acc)[V]) {
  constexpr int kBatch = 8;
  for (int b = 0; b < count; b += kBatch) {
    Vec<T, V> x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (b + i < count) x[i] = *reinterpret_cast<const Vec<T, V>*>(dy + static_cast<int64_t>(at[b + i]) * stride);
      else x[i].zero();
    }
    float part[V] = {};  // sums of sums: a chain of 8 + count / 8 additions
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (b + i >= count) break;
      float r[V];
      x[i].get(r);
#pragma unroll
      for (int k = 0; k < V; ++k) part[k] += r[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += part[k];
  }
}

template <typename T, typename TO, int V, bool Add>
__global__ void __launch_bounds__(kShortThreads)
    short_kernel(const __grid_constant__ KeySource src, int n, int64_t share, const T* __restrict__ dy, int64_t stride,
                 int d, float scale, TO* __restrict__ dw, int* err) {
  __shared__ uint32_t keys[kShortList], list[kShortList];
  __shared__ uint32_t flags[Add ? 1 : kShortFlags];
  __shared__ float meet[kShortWarps][32 * V];
  __shared__ int counts[kShortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t none = static_cast<uint32_t>(src.vocab);
  for (int i = threadIdx.x; i < n; i += kShortThreads) keys[i] = load_item(src, i, blockIdx.x == 0 ? err : nullptr).x;
  if constexpr (!Add) {
    for (int i = threadIdx.x; i < kShortFlags; i += kShortThreads) flags[i] = 0;
  }
  __syncthreads();
  if constexpr (!Add) {
    const int64_t first = blockIdx.x * share, left = src.vocab - first;
    const int rows = static_cast<int>(left < share ? (left > 0 ? left : 0) : share);
    for (int i = threadIdx.x; i < n; i += kShortThreads) {
      const int64_t at = static_cast<int64_t>(keys[i]) - first;
      if (at >= 0 && at < rows) atomicOr(&flags[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    const float zeros[V] = {};
    for (int r = warp; r < rows; r += kShortWarps) {
      if (flags[r >> 5] >> (r & 31) & 1u) continue;
      for (int col = lane * V; col < d; col += 32 * V) store_vec<TO, V>(dw + (first + r) * d + col, zeros);
    }
  }
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const uint32_t key = keys[i];
    if (key == none) continue;
    bool seen = false;
    for (int j = threadIdx.x; j < i; j += kShortThreads) seen |= keys[j] == key;
    if (__syncthreads_or(seen)) continue;
    // the positions of the token from here on, in order: warps take neighbouring segments of them
    const int segment = ((n - i + kShortWarps - 1) / kShortWarps + 31) / 32 * 32;
    const int from = i + warp * segment, to = from + segment < n ? from + segment : n;
    int count = 0;
    for (int j = from; j < to; j += 32) count += __popc(__ballot_sync(0xffffffffu, j + lane < to && keys[j + lane] == key));
    if (lane == 0) counts[warp] = count;
    __syncthreads();
    int place = 0, whole = 0;
    for (int w = 0; w < kShortWarps; ++w) {
      place += w < warp ? counts[w] : 0;
      whole += counts[w];
    }
    for (int j = from; j < to; j += 32) {
      const bool mine = j + lane < to && keys[j + lane] == key;
      const unsigned all = __ballot_sync(0xffffffffu, mine);
      if (mine) list[place + __popc(all & ((1u << lane) - 1))] = static_cast<uint32_t>(j + lane);
      place += __popc(all);
    }
    __syncthreads();
    TO* out = dw + static_cast<int64_t>(key) * d;
    if (whole <= kShortSerial) {
      for (int col = threadIdx.x * V; col < d; col += kShortThreads * V) {
        float acc[V] = {};
        add_rows<T, V>(list, whole, dy + col, stride, acc);
        write_row<TO, V, Add>(out + col, acc, scale);
      }
    } else {
      const int part = (whole + kShortWarps - 1) / kShortWarps, start = warp * part < whole ? warp * part : whole;
      const int mine = start + part < whole ? part : whole - start;
      for (int base = 0; base < d; base += 32 * V) {
        const int col = base + lane * V;
        float acc[V] = {};
        if (col < d) add_rows<T, V>(list + start, mine, dy + col, stride, acc);
#pragma unroll
        for (int k = 0; k < V; ++k) meet[warp][k * 32 + lane] = acc[k];
        __syncthreads();
        if (warp == 0 && col < d) {
#pragma unroll
          for (int k = 0; k < V; ++k)
            for (int w = 1; w < kShortWarps; ++w) acc[k] += meet[w][k * 32 + lane];
          write_row<TO, V, Add>(out + col, acc, scale);
        }
        __syncthreads();
      }
    }
    __syncthreads();  // list and counts are free again
  }
}

template <typename T, typename TO, int V>
int launch_short(const KeySource& src, int64_t n, const void* dy, int64_t stride, int d, float scale, bool accumulate,
                 void* dw, int64_t grid, int64_t share, int* err, cudaStream_t st) {
  const auto kernel = accumulate ? short_kernel<T, TO, V, true> : short_kernel<T, TO, V, false>;
  kernel<<<static_cast<unsigned>(grid), kShortThreads, 0, st>>>(src, static_cast<int>(n), share, static_cast<const T*>(dy),
                                                                stride, d, scale, static_cast<TO*>(dw), err);
  note_launch();
  OPUS_CUDA_TRY(cudaGetLastError());
  return OPUS_OK;
}

template <typename T, typename TO>
int launch_short_by_width(bool vec, const KeySource& src, int64_t n, const void* dy, int64_t stride, int d, float scale,
                          bool accumulate, void* dw, int64_t grid, int64_t share, int* err, cudaStream_t st) {
  return vec ? launch_short<T, TO, 16 / sizeof(TO)>(src, n, dy, stride, d, scale, accumulate, dw, grid, share, err, st)
             : launch_short<T, TO, 1>(src, n, dy, stride, d, scale, accumulate, dw, grid, share, err, st);
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

// Whether the `bytes` bytes at p share one with `rows` rows of d elements of `size` bytes, row_stride elements apart
// from q on.
bool overlaps(const void* p, int64_t bytes, const void* q, int64_t rows, int64_t d, int64_t row_stride, int size) {
  const int64_t from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q));
  const int64_t run = d * size, stride = std::min(row_stride, int64_t{1} << 56) * size;  // no address is that far away
  const int64_t row = from < run ? 0 : (from - run) / stride + 1;  // the first that ends behind p
  return row < rows && row * stride < from + bytes;
}

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
  const int size = dtype_bytes(dtype);
  if (overlaps(out, n * d * size, weight, vocab, d, row_stride, size) ||
      overlaps(out, n * d * size, tokens, 1, n, n, token_bits / 8))
    return set_error(OPUS_ERR_INVALID, "embedding: out overlaps what is read");
  int* err = token_error_word();
  if (err == nullptr) return set_error(OPUS_ERR_CUDA, "device error word unavailable");
  const int V = 16 / dtype_bytes(dtype);
  const bool vec = d % V == 0 && row_stride % V == 0 && aligned(weight, 16) && aligned(out, 16);
  const int wide = token_bits == 64;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == OPUS_DTYPE_F32)
    return launch_lookup_by_width<float>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
  if (dtype == OPUS_DTYPE_F16)
    return launch_lookup_by_width<__half>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
  return launch_lookup_by_width<__nv_bfloat16>(tokens, wide, n, weight, vocab, row_stride, d, scale, out, vec, err, st);
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
  const int64_t whole = vocab * d * dtype_bytes(out_dtype);
  if (overlaps(grad_weight, whole, grad_out, n, d, row_stride, dtype_bytes(grad_dtype)) ||
      overlaps(grad_weight, whole, tokens, 1, n, n, token_bits / 8))
    return set_error(OPUS_ERR_INVALID, "embedding_grad: grad_weight overlaps what is read");
  int* err = token_error_word();
  if (err == nullptr) return set_error(OPUS_ERR_CUDA, "device error word unavailable");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const KeySource src{tokens, nullptr, token_bits == 64, vocab, padding_idx};
  const int64_t zero_bytes = accumulate ? 0 : whole;
  const bool f32_out = out_dtype == OPUS_DTYPE_F32;
  const int V = 16 / (f32_out ? 4 : dtype_bytes(grad_dtype));
  const bool vec = d % V == 0 && row_stride % V == 0 && aligned(grad_out, V * dtype_bytes(grad_dtype)) &&
                   aligned(grad_weight, V * dtype_bytes(out_dtype));
  const int64_t grid = static_cast<int64_t>(sm_count()) * kShortBlocksPerSm, share = (vocab + grid - 1) / grid;
  const int64_t slabs = (d + 32 * (vec ? V : 1) - 1) / (32 * (vec ? V : 1));
  if (n <= kShortList && (n <= kShortSerial || (n + 63) / 64 * slabs <= kShortWork) && share <= kShortFlags * 32) {
    const auto run = grad_dtype == OPUS_DTYPE_F32   ? launch_short_by_width<float, float>
                     : grad_dtype == OPUS_DTYPE_F16 ? (f32_out ? launch_short_by_width<__half, float> : launch_short_by_width<__half, __half>)
                     : f32_out                      ? launch_short_by_width<__nv_bfloat16, float>
                                                    : launch_short_by_width<__nv_bfloat16, __nv_bfloat16>;
    return run(vec, src, n, grad_out, row_stride, d, scale, accumulate != 0, grad_weight, grid, share, err, st);
  }
  rc = p.cluster ? launch_cluster_sort(p, src, n, ws, grad_weight, zero_bytes, err, st)
                 : launch_global_sort(p, src, n, ws, grad_weight, zero_bytes, err, st);
  if (rc) return rc;
  if (grad_dtype == OPUS_DTYPE_F32)
    return launch_sums_by_width<float, float>(vec, p, n, vocab, grad_out, row_stride, d, scale, accumulate,
                                              grad_weight, ws, st);
  if (grad_dtype == OPUS_DTYPE_F16) {
    if (f32_out)
      return launch_sums_by_width<__half, float>(vec, p, n, vocab, grad_out, row_stride, d, scale,
                                                 accumulate, grad_weight, ws, st);
    return launch_sums_by_width<__half, __half>(vec, p, n, vocab, grad_out, row_stride, d, scale,
                                                accumulate, grad_weight, ws, st);
  }
  if (f32_out)
    return launch_sums_by_width<__nv_bfloat16, float>(vec, p, n, vocab, grad_out, row_stride, d, scale,
                                                      accumulate, grad_weight, ws, st);
  return launch_sums_by_width<__nv_bfloat16, __nv_bfloat16>(vec, p, n, vocab, grad_out, row_stride, d, scale,
                                                            accumulate, grad_weight, ws, st);
}
