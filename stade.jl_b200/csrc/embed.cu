// embed and embed_b: lookup of table rows with a scale, and the table's
// gradient by sorted ids.
//
//   v = ids[s] - base;  y[s, :] = scale w[v, :]   (0 <= v < n_v)
//   wb[v, :] += scale sum over the s with ids[s] - base == v, in increasing s, of yb[s, :]
//
// A negative v is padding: its row of y is zero and it adds to no row of the
// gradient. v >= n_v is treated the same and sets the device error word.
//
// The reverse sweep sorts (id, position) by id with a stable radix sort, so
// every table row's positions lie side by side in increasing order; sums of a
// row then need no atomics and always run in the same order.
//
// The lookup is bound by memory: 32768 rows of 1024 bf16 in 20.6 us, 0.99 of the
// measured copy rate by the bytes moved. The gradient of the same rows into a
// table of 50021 (205 MB of Float32) takes 65 us, 41 by its bytes: the sort, with
// the clearing beside it (34 us under the profiler), the sums (21 us) and the
// parts' join (11 us) wait for one another. Past 65,536 positions the sort no
// longer fits one cluster and takes five launches or more, whose digit counts one
// block scans: 65536 x 256 bf16 into 50021 rows 67 us, 65537 83, 262144 198 (28 by
// bytes), 1048576 x 64 639.

#include <cooperative_groups.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "token_ops.cuh"

namespace stade {
namespace {

__device__ int g_embed_error = 0;

constexpr int kThreads = 256;

// Whether an id is in the table; below base it is padding, past the table an
// error. Compared before the difference, which can pass 64 bits.
__device__ __forceinline__ bool in_table(int64_t id, int64_t base, int64_t n_v, bool* past) {
  const bool in = (uint64_t)id - (uint64_t)base < (uint64_t)n_v;
  *past = id >= base && !in;
  return id >= base && in;
}

// A warp takes kFwdRows consecutive positions: their ids first, then column by
// column one vector of each row, so that several rows' reads are in flight.
constexpr int kFwdRows = 4;

template <class T, int VEC>
__global__ void __launch_bounds__(kThreads)
embed_fwd_kernel(const T* __restrict__ w, const int64_t* __restrict__ ids, T* __restrict__ y,
                 acc_t<T> scale, int64_t base, int64_t n_s, int64_t n_v, int n_d) {
  using V = Vec<T, VEC>;
  const int lane = threadIdx.x & 31, slots = n_d / VEC;
  const int64_t s0 = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kFwdRows;
  if (s0 >= n_s) return;
  const V* row[kFwdRows];
  bool ok[kFwdRows], error = false;
#pragma unroll
  for (int q = 0; q < kFwdRows; ++q) {
    const int64_t id = s0 + q < n_s ? ids[s0 + q] : INT64_MIN;
    bool past;
    ok[q] = in_table(id, base, n_v, &past);
    error |= past;
    row[q] = reinterpret_cast<const V*>(w + (ok[q] ? id - base : 0) * n_d);
  }
  if (error) g_embed_error = 1;
  const int n = (int)min((int64_t)kFwdRows, n_s - s0);
  V* out = reinterpret_cast<V*>(y + s0 * n_d);
  for (int j = lane; j < slots; j += 32) {
    V r[kFwdRows];
#pragma unroll
    for (int q = 0; q < kFwdRows; ++q)
      if (ok[q]) r[q] = row[q][j];
#pragma unroll
    for (int q = 0; q < kFwdRows; ++q)
      if (q < n) {
        V o;
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          o.v[k] = round_to<T>(ok[q] ? scale * load_acc<T>(r[q].v[k]) : acc_t<T>(0));
        out[(int64_t)q * slots + j] = o;
      }
  }
}

// ---- stable radix sort of (key, position) -------------------------------------
// key = v, or n_v for padding. A pass sorts by one digit of at most 9 bits:
// counts per block, then a scatter in which each warp walks its own stretch of
// the block's elements in order, so equal keys keep their order. Up to
// kSmallSort elements one block does every pass in shared memory. The digit
// counts of the later passes are added up by the scatter before (whole
// numbers, so their order does not matter).
constexpr int kMaxBins = 512;
constexpr int kWarps = 8;
constexpr int kWarpItems = 128;
constexpr int kChunk = kWarps * kWarpItems;   // elements of one block
constexpr int kFusedScan = 64;                // blocks up to which a scatter adds the counts itself
constexpr int kSmallSort = 4096;

struct SortIn {
  const int64_t* ids;      // first pass: keys from the ids, positions 0 .. n - 1
  const uint32_t* keys;    // later passes
  const uint32_t* pos;
  int64_t base, n_v;
};
__device__ __forceinline__ uint32_t id_key(const SortIn& in, int64_t i) {
  const int64_t id = in.ids[i];
  bool past;
  const bool ok = in_table(id, in.base, in.n_v, &past);
  if (past) g_embed_error = 1;
  return (uint32_t)(ok ? id - in.base : in.n_v);
}
__device__ __forceinline__ uint32_t sort_key(const SortIn& in, int64_t i) {
  return in.ids ? id_key(in, i) : in.keys[i];
}

// Digit counts per block: [block][digit], which every block of the scatter reads
// through, or [digit][block] for the scan of many blocks.
__device__ __forceinline__ int64_t count_at(int digit, int block, int bins, int blocks,
                                            bool by_digit) {
  return by_digit ? (int64_t)digit * blocks + block : (int64_t)block * bins + digit;
}

// The sort keeps a few dozen blocks busy for some 30 us; the rest of the GPU
// meanwhile clears the gradient (when it is stored, not added to), so that the
// sums write only the rows that have positions. A kernel's blocks past `first`
// clear one part of it.
struct Fill {
  int4* p;              // 16-byte pieces, then single bytes up to `bytes`
  int64_t bytes;
  int part, parts;
};
__device__ __forceinline__ bool fill_block(const Fill& f, int first) {
  if ((int)blockIdx.x < first) return false;
  const int64_t n = f.bytes / 16, a = n * f.part / f.parts, z = n * (f.part + 1) / f.parts;
  const int64_t step = (int64_t)(gridDim.x - first) * blockDim.x;
  const int64_t t = (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x;
  int64_t i = a + t;
  for (; i + 3 * step < z; i += 4 * step)
#pragma unroll
    for (int u = 0; u < 4; ++u) f.p[i + u * step] = make_int4(0, 0, 0, 0);
  for (; i < z; i += step) f.p[i] = make_int4(0, 0, 0, 0);
  if (f.part == 0 && t < f.bytes % 16) reinterpret_cast<char*>(f.p + n)[t] = 0;
  return true;
}

// First pass: digit counts per block; zeroes the later passes' counts.
__global__ void __launch_bounds__(kThreads)
sort_count_kernel(SortIn in, int64_t n, int bins, int blocks, uint32_t* __restrict__ counts,
                  int64_t rest, bool by_digit, Fill fill) {
  __shared__ uint32_t h[kMaxBins];
  before_next();
  if (fill_block(fill, blocks)) return;
  for (int b = threadIdx.x; b < bins; b += kThreads) h[b] = 0;
  const int64_t mine = (int64_t)bins * blocks;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rest;
       i += (int64_t)blocks * kThreads)
    counts[mine + i] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kChunk, i1 = min(n, i0 + kChunk);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
    atomicAdd(&h[sort_key(in, i) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads)
    counts[count_at(b, blockIdx.x, bins, blocks, by_digit)] = h[b];
}

// Exclusive scan of one value per thread over the block; `sums`: 32 words.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t* sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    uint32_t a = lane < warps ? sums[lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, a, o);
      if (lane >= o) a += u;
    }
    sums[lane] = a;
  }
  __syncthreads();
  const uint32_t before = (warp ? sums[warp - 1] : 0u) + inc - x;
  *total = sums[warps - 1];
  __syncthreads();
  return before;
}

// exclusive scan in place, one block
__global__ void __launch_bounds__(1024) scan_kernel(uint32_t* __restrict__ v, int64_t n) {
  __shared__ uint32_t sums[32];
  uint32_t carry = 0;
  before_next();
  after_previous();
  for (int64_t i0 = 0; i0 < n; i0 += 1024) {
    const int64_t i = i0 + threadIdx.x;
    uint32_t total;
    const uint32_t before = block_exclusive(i < n ? v[i] : 0u, sums, &total);
    if (i < n) v[i] = carry + before;
    carry += total;
  }
}

// counts: digit counts per block (`scanned`: their exclusive scan); next: the
// next pass's counts, which this one adds up, or null.
__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(SortIn in, int64_t n, int shift, int bins, int blocks,
                    const uint32_t* __restrict__ counts, bool scanned, uint32_t* __restrict__ next,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, Fill fill) {
  __shared__ uint32_t h[kWarps][kMaxBins];
  __shared__ uint32_t start[kMaxBins];
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  before_next();
  if (fill_block(fill, blocks)) return;      // touches nothing of the kernel before
  for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&h[0][0])[b] = 0;
  after_previous();
  const int64_t w0 = (int64_t)blockIdx.x * kChunk + warp * kWarpItems;
  uint32_t key[kWarpItems / 32];
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u) {
    const int64_t i = w0 + u * 32 + lane;
    key[u] = i < n ? sort_key(in, i) : 0xffffffffu;
  }
  // where this block's elements of each digit begin
  if (scanned) {
    for (int b = threadIdx.x; b < bins; b += kThreads)
      start[b] = counts[count_at(b, blockIdx.x, bins, blocks, true)];
    __syncthreads();
  } else {
    uint32_t carry = 0;
    for (int b0 = 0; b0 < bins; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      uint32_t all = 0, before = 0;
      if (b < bins)
#pragma unroll 8
        for (int j = 0; j < blocks; ++j) {
          const uint32_t c = counts[count_at(b, j, bins, blocks, false)];
          all += c;
          if (j < (int)blockIdx.x) before += c;
        }
      uint32_t total;
      const uint32_t ahead = block_exclusive(all, sums, &total);
      if (b < bins) start[b] = carry + ahead + before;
      carry += total;
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u)
    if (w0 + u * 32 + lane < n) atomicAdd(&h[warp][(key[u] >> shift) & (bins - 1)], 1u);
  __syncthreads();
  // per digit: this block's start, then the warps one after the other
  for (int b = threadIdx.x; b < bins; b += kThreads) {
    uint32_t at = start[b];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = h[w][b];
      h[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u) {
    const int64_t i = w0 + u * 32 + lane;
    const bool in_range = i < n;
    const uint32_t bin = in_range ? (key[u] >> shift) & (bins - 1) : 0xffffffffu;
    const uint32_t peers = __match_any_sync(0xffffffffu, bin);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    uint32_t at = 0;
    if (in_range) at = h[warp][bin] + rank;
    __syncwarp();
    if (in_range && rank == 0) h[warp][bin] += __popc(peers);
    __syncwarp();
    if (in_range) {
      keys_out[at] = key[u];
      pos_out[at] = in.ids ? (uint32_t)i : in.pos[i];
      if (next)
        atomicAdd(&next[count_at((key[u] >> (shift + __popc(bins - 1))) & (bins - 1), at / kChunk,
                                 bins, blocks, scanned)], 1u);
    }
  }
}

// The whole sort for n <= kSmallSort in one block (the others clear).
constexpr int kSmallItems = 256;              // elements of a warp
constexpr int kSmallWarps = kSmallSort / kSmallItems;
constexpr int kSmallThreads = kSmallWarps * 32;
// A launch's shared memory, at most. The sorts' limits are set to these whatever
// a call needs: the limit is the kernel's, and a host thread with another size
// must not lower it between this call's setting and its launch.
constexpr int kSmallSmem = (2 * kSmallSort + kSmallWarps * kMaxBins) * 4;
__global__ void __launch_bounds__(kSmallThreads)
small_sort_kernel(SortIn in, int n, int passes, int bits, uint32_t* __restrict__ keys_out,
                  uint32_t* __restrict__ pos_out, Fill fill) {
  extern __shared__ uint32_t sm[];
  uint32_t* keys = sm;
  uint32_t* pos = sm + kSmallSort;
  uint32_t* h = sm + 2 * kSmallSort;             // [kSmallWarps][bins]
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << bits;
  before_next();
  if (fill_block(fill, 1)) return;
  const int w0 = warp * kSmallItems;
  uint32_t key[kSmallItems / 32], p[kSmallItems / 32];
#pragma unroll
  for (int u = 0; u < kSmallItems / 32; ++u) {
    const int i = w0 + u * 32 + lane;
    key[u] = i < n ? id_key(in, i) : 0xffffffffu;
    p[u] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int b = threadIdx.x; b < kSmallWarps * bins; b += kSmallThreads) h[b] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kSmallItems / 32; ++u)
      if (w0 + u * 32 + lane < n) atomicAdd(&h[warp * bins + ((key[u] >> shift) & (bins - 1))], 1u);
    __syncthreads();
    // one digit a thread (bins <= 512 threads), its warps one after the other
    uint32_t all = 0;
    if ((int)threadIdx.x < bins)
      for (int w = 0; w < kSmallWarps; ++w) all += h[w * bins + threadIdx.x];
    uint32_t total, at = block_exclusive(all, sums, &total);
    if ((int)threadIdx.x < bins)
      for (int w = 0; w < kSmallWarps; ++w) {
        const uint32_t c = h[w * bins + threadIdx.x];
        h[w * bins + threadIdx.x] = at;
        at += c;
      }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kSmallItems / 32; ++u) {
      const bool in_range = w0 + u * 32 + lane < n;
      const uint32_t bin = in_range ? (key[u] >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, bin);
      const int rank = __popc(peers & ((1u << lane) - 1u));
      uint32_t to = 0;
      if (in_range) to = h[warp * bins + bin] + rank;
      __syncwarp();
      if (in_range && rank == 0) h[warp * bins + bin] += __popc(peers);
      __syncwarp();
      if (in_range) {
        keys[to] = key[u];
        pos[to] = p[u];
      }
    }
    __syncthreads();
    if (pass + 1 < passes)
#pragma unroll
      for (int u = 0; u < kSmallItems / 32; ++u) {
        const int i = w0 + u * 32 + lane;
        if (i < n) key[u] = keys[i], p[u] = pos[i];
      }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSmallThreads) {
    keys_out[i] = keys[i];
    pos_out[i] = pos[i];
  }
}

// The whole sort for n up to kClusterSort in one cluster of kSortCtas blocks (the
// other clusters clear): each block holds its share of the keys in shared
// memory, a pass adds the blocks' digit counts up over distributed shared
// memory and stores every key where it belongs, in whichever block that is.
// The embedding gradient of 32768 x 1024 bf16 into 50021 rows takes 85 us with
// three launches for the sort, 65 us so; the sort alone 25 us, with the clearing
// of 205 MB beside it 34.
constexpr int kSortCtas = 8;
constexpr int kSortWarps = 32;
constexpr int kLaneItems = 8;               // keys a lane holds, at most
constexpr int kClusterSort = kSortCtas * kSortWarps * 32 * kLaneItems;
constexpr int kClusterSmem = (2 * kSortWarps * 32 * kLaneItems + kSortWarps * kMaxBins) * 4;

__global__ void __launch_bounds__(32 * kSortWarps)
cluster_sort_kernel(SortIn in, int n, int passes, int bits, int lane_items,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, Fill fill) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t total[kMaxBins];
  __shared__ uint32_t sums[32];
  before_next();
  if (fill_block(fill, kSortCtas)) return;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << bits;
  const int per_warp = 32 * lane_items, share = kSortWarps * per_warp;
  uint32_t* keys = sm;
  uint32_t* pos = sm + share;
  uint32_t* h = sm + 2 * share;               // [kSortWarps][bins]
  const int mine = warp * per_warp;           // of the block's share
  const int valid = n - rank * share;         // keys of the block's share that exist
  uint32_t key[kLaneItems], p[kLaneItems];
#pragma unroll
  for (int u = 0; u < kLaneItems; ++u) {
    const int i = mine + u * 32 + lane;
    const bool has = u < lane_items && i < valid;
    key[u] = has ? id_key(in, (int64_t)rank * share + i) : 0xffffffffu;
    p[u] = rank * share + i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int b = threadIdx.x; b < kSortWarps * bins; b += 32 * kSortWarps) h[b] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kLaneItems; ++u)
      if (u < lane_items && mine + u * 32 + lane < valid)
        atomicAdd(&h[warp * bins + ((key[u] >> shift) & (bins - 1))], 1u);
    __syncthreads();
    if ((int)threadIdx.x < bins) {
      uint32_t t = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) t += h[w * bins + threadIdx.x];
      total[threadIdx.x] = t;
    }
    cluster.sync();       // every block's counts are there, and its keys in registers
    uint32_t all = 0, before = 0;
    if ((int)threadIdx.x < bins) {
      uint32_t c[kSortCtas];
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) c[r] = *cluster.map_shared_rank(&total[threadIdx.x], r);
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) {
        all += c[r];
        if (r < rank) before += c[r];
      }
    }
    uint32_t sum;
    const uint32_t ahead = block_exclusive(all, sums, &sum);
    if ((int)threadIdx.x < bins) {
      uint32_t at = ahead + before;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = h[w * bins + threadIdx.x];
        h[w * bins + threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kLaneItems; ++u) {
      const bool in_range = u < lane_items && mine + u * 32 + lane < valid;
      const uint32_t bin = in_range ? (key[u] >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, bin);
      const int before_me = __popc(peers & ((1u << lane) - 1u));
      uint32_t to = 0;
      if (in_range) to = h[warp * bins + bin] + before_me;
      __syncwarp();
      if (in_range && before_me == 0) h[warp * bins + bin] += __popc(peers);
      __syncwarp();
      if (in_range) {
        const uint32_t owner = to / share, at = to - owner * share;
        *cluster.map_shared_rank(&keys[at], owner) = key[u];
        *cluster.map_shared_rank(&pos[at], owner) = p[u];
      }
    }
    cluster.sync();
#pragma unroll
    for (int u = 0; u < kLaneItems; ++u) {
      const int i = mine + u * 32 + lane;
      if (u < lane_items && i < valid) key[u] = keys[i], p[u] = pos[i];
    }
  }
#pragma unroll
  for (int u = 0; u < kLaneItems; ++u) {
    const int i = mine + u * 32 + lane;
    if (u < lane_items && i < valid) {
      keys_out[(int64_t)rank * share + i] = key[u];
      pos_out[(int64_t)rank * share + i] = p[u];
    }
  }
}

// ---- sums of rows ----------------------------------------------------------------
// After the sort a table row's positions lie side by side: a run. A warp takes
// a window of `width` sorted positions and kCols vectors a lane of their
// columns, whatever runs lie in it, so all warps read the same amount; a run
// inside the window is written where it ends, one that crosses the window's
// edges leaves its part (head: begun before the window; tail: begun in it) and
// join_kernel adds a run's parts in order. The id that takes a tenth of a batch
// costs what its rows cost.
struct SumArgs {
  const uint32_t *keys, *pos;
  const void* yb;
  void *wb, *part;       // part: [window][head, tail][n_d]
  double scale;
  int64_t n, n_v;
  int n_d, width, chunks;
  bool add;
};

// A vector of VEC columns is 16 bytes of the gradient: 4 Float32 (read as 8 or
// 16 bytes of yb), 2 Float64, or single columns where rows do not allow it.
template <class A, int VEC>
__device__ __forceinline__ void put(A* p, const A (&v)[VEC], A scale, bool add) {
  Vec<A, VEC> o;
  if (add) o = *reinterpret_cast<const Vec<A, VEC>*>(p);
#pragma unroll
  for (int k = 0; k < VEC; ++k) o.v[k] = add ? o.v[k] + v[k] * scale : v[k] * scale;
  *reinterpret_cast<Vec<A, VEC>*>(p) = o;
}

constexpr int kCols = 4;         // vectors of a lane that a warp sums at once
constexpr int kMaxWidth = 64;

template <class T, int VEC>
__global__ void __launch_bounds__(kThreads)
window_sum_kernel(SumArgs p) {
  using A = acc_t<T>;
  using V = Vec<T, VEC>;
  constexpr int kSpan = 32 * VEC * kCols, U = 4;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t win = item / p.chunks, p0 = win * p.width;
  if (p0 >= p.n) return;
  const int col = (int)(item % p.chunks) * kSpan + lane * VEC;
  before_next();
  after_previous();
  const int len = (int)min((int64_t)p.width, p.n - p0);
  const uint32_t none = (uint32_t)p.n_v;
  // this window's keys and positions, two a lane, and the keys beside it
  uint32_t key[2], at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool in = 32 * h + lane < len;
    key[h] = in ? p.keys[p0 + 32 * h + lane] : none;
    at[h] = in ? p.pos[p0 + 32 * h + lane] : 0u;
  }
  const uint32_t before = p0 > 0 ? p.keys[p0 - 1] : 0xffffffffu;
  const uint32_t after = p0 + len < p.n ? p.keys[p0 + len] : 0xffffffffu;
  auto key_of = [&](int i) {
    return __shfl_sync(0xffffffffu, i < 32 ? key[0] : key[1], i & 31);
  };
  const T* yb = (const T*)p.yb;
  const A scale = (A)p.scale;
  // sums in pairs (one value a vector where rows allow no more)
  constexpr int NP = VEC > 1 ? VEC / 2 : 1;
  Pair<A> acc[kCols][NP];
  bool has[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    has[c] = col + c * 32 * VEC < p.n_d;
#pragma unroll
    for (int j = 0; j < NP; ++j) acc[c][j] = both(A(0));
  }
  const T* mine = yb + col;
  int first = 0;                       // where the current run begins in the window
  for (int i0 = 0; i0 < len; i0 += U) {
    if (key_of(i0) == none) break;     // padding sorts last
    V r[U][kCols];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      const uint32_t row = __shfl_sync(0xffffffffu, i < 32 ? at[0] : at[1], i & 31);
      if (i < len) {
        const T* q = mine + (int64_t)row * p.n_d;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          if (has[c]) r[u][c] = *reinterpret_cast<const V*>(q + c * 32 * VEC);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      const uint32_t k = key_of(i < len ? i : 0), k1 = key_of(i + 1 < len ? i + 1 : 0);
      if (i >= len || k == none) break;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if constexpr (VEC > 1)
            acc[c][j] = add2(acc[c][j], widen2(reinterpret_cast<const Vec<T, 2>*>(&r[u][c])[j]));
          else
            acc[c][j] = Pair<A>(acc[c][j].lo() + load_acc<T>(r[u][c].v[0]), A(0));
        }
      const bool edge = i + 1 == len;
      if (!edge && k1 == k) continue;
      // the run, or the window's share of it, ends here
      const bool begun = first > 0 || before != k, ended = !edge || after != k;
      const bool whole = begun && ended;
      A* o = whole ? (A*)p.wb + (int64_t)k * p.n_d
                   : (A*)p.part + (2 * win + (begun ? 1 : 0)) * p.n_d;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        if (has[c]) {
          A v[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[j] = j % 2 ? acc[c][j / 2].hi() : acc[c][j / 2].lo();
          put<A, VEC>(o + col + c * 32 * VEC, v, whole ? scale : A(1), whole && p.add);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) acc[c][j] = both(A(0));
      }
      first = i + 1;
    }
  }
}

// A run that begins in a window and goes on past it: its tail there, then the
// heads of the windows that follow, in order.
template <class A, int VEC>
__global__ void __launch_bounds__(kThreads)
join_kernel(SumArgs p) {
  constexpr int kSpan = 32 * VEC, U = 8;
  const int lane = threadIdx.x & 31;
  const int chunks = (p.n_d + kSpan - 1) / kSpan;
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t win = item / chunks, p1 = (win + 1) * p.width;
  if (p1 >= p.n) return;
  after_previous();
  const int64_t p0 = win * p.width;
  const uint32_t k = p.keys[p1 - 1], next = p.keys[p1];
  const uint32_t before = p0 > 0 ? p.keys[p0 - 1] : 0xffffffffu;
  // nothing goes on past the window, or what does has begun before it
  if (k == (uint32_t)p.n_v || next != k || before == k) return;
  // heads: of window win + 1 + j while its first key is k
  int64_t heads = 0;
  for (;;) {
    const int64_t q = p1 + (heads + lane) * p.width;
    const uint32_t same = __ballot_sync(0xffffffffu, q < p.n && p.keys[min(q, p.n - 1)] == k);
    const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
    heads += run;
    if (run < 32) break;
  }
  const int col = (int)(item % chunks) * kSpan + lane * VEC;
  if (col >= p.n_d) return;
  const A* part = (const A*)p.part + col;
  using V = Vec<A, VEC>;
  const V t = *reinterpret_cast<const V*>(part + (2 * win + 1) * p.n_d);
  A acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = t.v[j];
  for (int64_t h = 0; h < heads; h += U) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u < heads)
        r[u] = *reinterpret_cast<const V*>(part + 2 * (win + 1 + h + u) * p.n_d);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u < heads)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += r[u].v[j];
  }
  put<A, VEC>((A*)p.wb + (int64_t)k * p.n_d + col, acc, (A)p.scale, p.add);
}

struct SortPlan {
  int passes, bits;      // digits, bits of a digit
  int64_t blocks;
  int64_t counts() const { return (int64_t)passes * (blocks << bits); }
};
SortPlan sort_plan(int64_t n_s, int64_t n_v) {
  int total = 1;
  while ((int64_t(1) << total) <= n_v) ++total;   // keys 0 .. n_v
  SortPlan p;
  p.passes = (total + 8) / 9;
  p.bits = (total + p.passes - 1) / p.passes;
  p.blocks = (n_s + kChunk - 1) / kChunk;
  return p;
}

// Calls f(VEC): 16 bytes of the 16-bit type (forward) or of the gradient
// (reverse) where alignment allows it, else 4 bytes forward, else one value.
template <class T, class F>
stade_status with_fwd_vec(int align, F&& f) {
  using std::integral_constant;
  if (align >= 16) return f(integral_constant<int, 16 / (int)sizeof(T)>{});
  if constexpr (sizeof(T) == 2)
    if (align >= 4) return f(integral_constant<int, 2>{});
  return f(integral_constant<int, 1>{});
}
template <class T, class F>
stade_status with_sum_vec(int align_t, int align_p, F&& f) {
  using std::integral_constant;
  constexpr int W = 16 / (int)sizeof(acc_t<T>);
  if (align_t >= W * (int)sizeof(T) && align_p >= 16) return f(integral_constant<int, W>{});
  return f(integral_constant<int, 1>{});
}
// Positions of a window: as many as leave eight warps an SM something to do (a
// warp's four rows in flight are 4 KB of 16-bit values; narrower windows leave
// more parts to join: 104 us against 96 with 24 warps an SM, 32768 x 1024 bf16).
int window_width(int64_t n_s, int64_t chunks) {
  int w = kMaxWidth;
  while (w > 8 && n_s * chunks / w < 148 * 8) w /= 2;
  return w;
}

struct Scratch {
  uint32_t *keys[2], *pos[2], *counts;
  double* part;
};
// S: Sizer or Carver
template <class S>
Scratch layout(S& z, int64_t n_s, int64_t n_v, int64_t n_d) {
  Scratch s{};
  auto take = [&](auto** to, size_t n) {
    using E = std::remove_pointer_t<std::remove_pointer_t<decltype(to)>>;
    if constexpr (std::is_same<S, Sizer>::value) z.template take<E>(n);
    else *to = z.template take<E>(n);
  };
  for (int i = 0; i < 2; ++i) {
    take(&s.keys[i], n_s);
    take(&s.pos[i], n_s);
  }
  take(&s.counts, sort_plan(n_s, n_v).counts());
  // the widest windows' parts, or the narrowest's of a short batch
  const int64_t wins =
      std::min<int64_t>((n_s + 7) / 8, (n_s + kMaxWidth - 1) / kMaxWidth + 148 * 16);
  take(&s.part, 2 * wins * n_d);
  return s;
}

stade_status check_sizes(const char* who, int dtype, int64_t n_s, int64_t n_v, int64_t n_d) {
  STADE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  STADE_REQUIRE(n_s >= 0 && n_v >= 0 && n_d >= 0, "%s: negative size", who);
  int64_t t;
  STADE_REQUIRE(n_s < (int64_t(1) << 31) && n_v < (int64_t(1) << 31) - 1 &&
                    n_d < (int64_t(1) << 31) && mul_ok(n_s, n_d, &t) && mul_ok(n_v, n_d, &t),
                "%s: size overflow", who);
  return STADE_OK;
}

}  // namespace

int embed_take_error() {
  int host = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&host, g_embed_error, sizeof(int)) != cudaSuccess) return -1;
  if (host) cudaMemcpyToSymbol(g_embed_error, &zero, sizeof(int));
  return host;
}

}  // namespace stade

using namespace stade;

extern "C" stade_status stade_embed(int dtype, const void* w, const int64_t* ids, void* y,
                                    double scale, int64_t base, int64_t n_s, int64_t n_v,
                                    int64_t n_d, const stade_opts* opts) {
  stade_status st = check_sizes("embed", dtype, n_s, n_v, n_d);
  if (st != STADE_OK) return st;
  if (n_s == 0 || n_d == 0) return STADE_OK;
  STADE_REQUIRE((w || n_v == 0) && ids && y, "embed: null array argument");
  cudaStream_t s = stream_of(opts);
  PhaseScope ph("embed", s);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return with_fwd_vec<T>(row_align(n_d * sizeof(T), {w, y}), [&](auto vec) {
      embed_fwd_kernel<T, decltype(vec)::value>
          <<<ceil_div_u(n_s, kFwdRows * (kThreads / 32)), kThreads, 0, s>>>(
              (const T*)w, ids, (T*)y, (acc_t<T>)scale, base, n_s, n_v, (int)n_d);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  });
}

extern "C" size_t stade_embed_b_workspace(int64_t n_s, int64_t n_v, int64_t n_d) {
  if (n_s <= 0 || n_v <= 0 || n_d <= 0) return 0;
  Sizer z;
  layout(z, n_s, n_v, n_d);
  return z.bytes();
}

extern "C" stade_status stade_embed_b(int dtype, void* wb, const int64_t* ids, void* yb,
                                      double scale, int64_t base, int64_t n_s, int64_t n_v,
                                      int64_t n_d, const stade_opts* opts) {
  stade_status st = check_sizes("embed_b", dtype, n_s, n_v, n_d);
  if (st != STADE_OK) return st;
  cudaStream_t s = stream_of(opts);
  const bool add = accumulates(opts);
  const size_t acc_size = dtype == STADE_F64 ? 8 : 4;
  if (n_d == 0) return STADE_OK;
  STADE_REQUIRE((wb || n_v == 0) && ((ids && yb) || n_s == 0), "embed_b: null array argument");
  if (n_v > 0 && n_s == 0) {
    if (!add) STADE_CUDA(cudaMemsetAsync(wb, 0, (size_t)n_v * n_d * acc_size, s));
    return STADE_OK;
  }
  PhaseScope ph("embed_b", s);
  if (n_v > 0) {
    void* ws = nullptr;
    st = get_workspace(opts, stade_embed_b_workspace(n_s, n_v, n_d), &ws);
    if (st != STADE_OK) return st;
    Carver c(ws);
    const Scratch sc = layout(c, n_s, n_v, n_d);
    const SortPlan p = sort_plan(n_s, n_v);
    const int bins = 1 << p.bits;
    st = with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      using A = acc_t<T>;
      return with_sum_vec<T>(row_align(n_d * sizeof(T), {yb}), row_align(n_d * sizeof(A), {wb}),
                             [&](auto vec) -> stade_status {
        constexpr int VEC = decltype(vec)::value;
        const int chunks = (int)((n_d + 32 * VEC * kCols - 1) / (32 * VEC * kCols));
        const int64_t bytes = n_v * n_d * (int64_t)sizeof(A);
        const bool whole = row_align(16, {wb}) == 16;     // 16-byte pieces can clear it
        if (!add && !whole) STADE_CUDA(cudaMemsetAsync(wb, 0, bytes, s));
        const int clearers =
            add || !whole ? 0 : (int)std::min<int64_t>(148 * 4, bytes / 16384 + 1);
        Fill fill{static_cast<int4*>(wb), bytes, 0, 1};
        int last = 0;
        if (n_s <= kSmallSort) {
          const size_t smem = (2 * kSmallSort + (size_t)kSmallWarps * bins) * 4;
          STADE_CUDA(cudaFuncSetAttribute(small_sort_kernel,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallSmem));
          small_sort_kernel<<<1 + clearers, kSmallThreads, smem, s>>>(
              SortIn{ids, nullptr, nullptr, base, n_v}, (int)n_s, p.passes, p.bits, sc.keys[0],
              sc.pos[0], fill);
          STADE_CHECK_LAUNCH();
        } else if (n_s <= kClusterSort) {
          const int lane_items = (int)((n_s + kClusterSort / kLaneItems - 1) /
                                       (kClusterSort / kLaneItems));
          const size_t smem =
              (2 * (size_t)kSortWarps * 32 * lane_items + (size_t)kSortWarps * bins) * 4;
          STADE_CUDA(cudaFuncSetAttribute(cluster_sort_kernel,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, kClusterSmem));
          cudaLaunchConfig_t cfg = {};
          // clusters that clear: with the sort's no more than can be on the GPU at
          // once (two of eight blocks in each of eight groups of SMs), since one
          // that starts late would end late
          const int clearing = (std::min(clearers, kSortCtas * 14) + kSortCtas - 1) / kSortCtas;
          cfg.gridDim = dim3(kSortCtas * (1 + clearing));
          cfg.blockDim = dim3(32 * kSortWarps);
          cfg.dynamicSmemBytes = smem;
          cfg.stream = s;
          cudaLaunchAttribute attr[1];
          attr[0].id = cudaLaunchAttributeClusterDimension;
          attr[0].val.clusterDim.x = kSortCtas;
          attr[0].val.clusterDim.y = 1;
          attr[0].val.clusterDim.z = 1;
          cfg.attrs = attr;
          cfg.numAttrs = 1;
          STADE_CUDA(cudaLaunchKernelEx(&cfg, cluster_sort_kernel,
                                        SortIn{ids, nullptr, nullptr, base, n_v}, (int)n_s, p.passes,
                                        p.bits, lane_items, sc.keys[0], sc.pos[0], fill));
          count_launch();
        } else {
          const int64_t per_pass = p.blocks << p.bits;
          const bool scan = p.blocks > kFusedScan;
          fill.parts = p.passes + 1;
          for (int i = 0; i < p.passes; ++i) {
            const SortIn in{i == 0 ? ids : nullptr, sc.keys[(i + 1) & 1], sc.pos[(i + 1) & 1], base,
                            n_v};
            uint32_t* counts = sc.counts + i * per_pass;
            if (i == 0) {
              sort_count_kernel<<<(unsigned)p.blocks + clearers, kThreads, 0, s>>>(
                  in, n_s, bins, (int)p.blocks, counts, (p.passes - 1) * per_pass, scan, fill);
              STADE_CHECK_LAUNCH();
            }
            if (scan) {
              st = launch_next(scan_kernel, 1, 1024, 0, s, counts, per_pass);
              if (st != STADE_OK) return st;
            }
            fill.part = i + 1;
            st = launch_next(sort_scatter_kernel, (unsigned)p.blocks + clearers, kThreads, 0, s, in,
                             n_s, i * p.bits, bins, (int)p.blocks, counts, scan,
                             i + 1 < p.passes ? counts + per_pass : nullptr, sc.keys[i & 1],
                             sc.pos[i & 1], fill);
            if (st != STADE_OK) return st;
          }
          last = (p.passes - 1) & 1;
        }
        const int width = window_width(n_s, chunks);
        const SumArgs a{sc.keys[last], sc.pos[last], yb, wb, sc.part, scale, n_s, n_v, (int)n_d,
                        width, chunks, add};
        const int64_t wins = (n_s + width - 1) / width;
        st = launch_next(window_sum_kernel<T, VEC>, ceil_div_u(wins * chunks, kWarps), kThreads, 0,
                         s, a);
        if (st != STADE_OK || wins == 1) return st;
        const int64_t join_chunks = (n_d + 32 * VEC - 1) / (32 * VEC);
        return launch_next(join_kernel<A, VEC>, ceil_div_u((wins - 1) * join_chunks, kWarps),
                           kThreads, 0, s, a);
      });
    });
    if (st != STADE_OK) return st;
  }
  if (consumes(opts)) STADE_CUDA(cudaMemsetAsync(yb, 0, (size_t)n_s * n_d * dtype_size(dtype), s));
  return STADE_OK;
}
