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

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "token_ops.cuh"

namespace stade {
namespace {

__device__ int g_embed_error = 0;

constexpr int kThreads = 256;

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
  bool ok[kFwdRows];
#pragma unroll
  for (int q = 0; q < kFwdRows; ++q) {
    const int64_t v = s0 + q < n_s ? ids[s0 + q] - base : -1;
    ok[q] = v >= 0 && v < n_v;
    if (v >= n_v && lane == 0) g_embed_error = 1;
    row[q] = reinterpret_cast<const V*>(w + (ok[q] ? v : 0) * n_d);
  }
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
constexpr int kWarpItems = 256;
constexpr int kChunk = kWarps * kWarpItems;   // elements of one block
constexpr int kFusedScan = 64;                // blocks up to which a scatter adds the counts itself
constexpr int kSmallSort = 4096;

// ---- sums of rows ----------------------------------------------------------------
// After the sort a table row's positions lie side by side. Rows of up to kShort
// positions are summed by one warp; longer ones are cut into pieces of up to
// kPiece positions, a block each (its warps take an eighth of the piece one
// after the other's end), whose sums the last block of the row adds up in
// order. The id that takes a tenth of a batch then costs what its rows cost.
constexpr int kShort = 32;
constexpr int kPiece = 512;

struct Piece {
  uint32_t v, from, len, first, count;   // first piece of the row and how many it has
};

struct SortIn {
  const int64_t* ids;      // first pass: keys from the ids, positions 0 .. n - 1
  const uint32_t* keys;    // later passes
  const uint32_t* pos;
  int64_t base, n_v;
};
__device__ __forceinline__ uint32_t id_key(const SortIn& in, int64_t i) {
  const int64_t v = in.ids[i] - in.base;
  if (v >= in.n_v) g_embed_error = 1;
  return (uint32_t)(v >= 0 && v < in.n_v ? v : in.n_v);
}
__device__ __forceinline__ uint32_t sort_key(const SortIn& in, int64_t i) {
  return in.ids ? id_key(in, i) : in.keys[i];
}

// First pass: digit counts per block; zeroes the later passes' counts and the
// number of pieces.
__global__ void __launch_bounds__(kThreads)
sort_count_kernel(SortIn in, int64_t n, int bins, uint32_t* __restrict__ counts, int64_t rest,
                  uint32_t* __restrict__ n_pieces) {
  __shared__ uint32_t h[kMaxBins];
  for (int b = threadIdx.x; b < bins; b += kThreads) h[b] = 0;
  const int64_t mine = (int64_t)bins * gridDim.x;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rest;
       i += (int64_t)gridDim.x * kThreads)
    counts[mine + i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *n_pieces = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kChunk, i1 = min(n, i0 + kChunk);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
    atomicAdd(&h[sort_key(in, i) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads)
    counts[(int64_t)b * gridDim.x + blockIdx.x] = h[b];
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
sort_scatter_kernel(SortIn in, int64_t n, int shift, int bins, const uint32_t* __restrict__ counts,
                    bool scanned, uint32_t* __restrict__ next, uint32_t* __restrict__ keys_out,
                    uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t h[kWarps][kMaxBins];
  __shared__ uint32_t start[kMaxBins];
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = gridDim.x;
  for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&h[0][0])[b] = 0;
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
      start[b] = counts[(int64_t)b * blocks + blockIdx.x];
    __syncthreads();
  } else {
    uint32_t carry = 0;
    for (int b0 = 0; b0 < bins; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      uint32_t all = 0, before = 0;
      if (b < bins)
        for (int j = 0; j < blocks; ++j) {
          const uint32_t c = counts[(int64_t)b * blocks + j];
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
        atomicAdd(&next[(int64_t)((key[u] >> (shift + __popc(bins - 1))) & (bins - 1)) * blocks +
                        at / kChunk], 1u);
    }
  }
}

// The piece list of a row of more than kShort positions.
__device__ __forceinline__ void list_pieces(uint32_t v, uint32_t from, uint32_t to,
                                            uint32_t* n_pieces, Piece* pieces, uint32_t* joins,
                                            int chunks) {
  const uint32_t len = to - from, count = (len + kPiece - 1) / kPiece;
  const uint32_t first = atomicAdd(n_pieces, count);
  for (uint32_t p = 0; p < count; ++p)
    pieces[first + p] = Piece{v, from + p * kPiece, min((uint32_t)kPiece, len - p * kPiece), first,
                              count};
  for (int c = 0; c < chunks; ++c) joins[(int64_t)first * chunks + c] = 0;
}

// start[v] = number of sorted keys below v, v = 0 .. n_v, and the pieces of the
// long rows. One thread per position: it fills the gap of keys that end at its
// own, together with its warp where the gap is long.
template <class Keys>
__device__ __forceinline__ void row_starts(Keys keys, uint32_t n, uint32_t n_v, uint32_t i,
                                           uint32_t* start, uint32_t* n_pieces, Piece* pieces,
                                           uint32_t* joins, int chunks) {
  const int lane = threadIdx.x & 31;
  // keys key[i - 1] + 1 .. key[i] begin at i (i = n: up to n_v)
  const uint32_t lo = i == 0 ? 0u : i <= n ? keys(i - 1) + 1 : 1u;
  const uint32_t hi = i < n ? keys(i) : i == n ? n_v : 0u;
  const bool has = i <= n && lo <= hi;
  const bool wide = has && hi - lo >= 8;
  if (has && !wide)
    for (uint32_t v = lo; v <= hi; ++v) start[v] = i;
  uint32_t todo = __ballot_sync(0xffffffffu, wide);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const uint32_t a = __shfl_sync(0xffffffffu, lo, src), z = __shfl_sync(0xffffffffu, hi, src);
    const uint32_t at = __shfl_sync(0xffffffffu, i, src);
    for (uint64_t v = (uint64_t)a + lane; v <= z; v += 32) start[v] = at;
  }
  if (has && i < n && hi < n_v && i + kShort < n && keys(i + kShort) == hi) {
    uint32_t a = i + kShort, z = n;          // keys(a) == hi, the run ends in (a, z]
    while (z - a > 1) {
      const uint32_t mid = a + (z - a) / 2;
      if (keys(mid) == hi) a = mid;
      else z = mid;
    }
    list_pieces(hi, i, z, n_pieces, pieces, joins, chunks);
  }
}

__global__ void __launch_bounds__(kThreads)
row_start_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t n_v,
                 uint32_t* __restrict__ start, uint32_t* __restrict__ n_pieces,
                 Piece* __restrict__ pieces, uint32_t* __restrict__ joins, int chunks) {
  row_starts([&](uint32_t i) { return keys[i]; }, n, n_v, blockIdx.x * kThreads + threadIdx.x,
             start, n_pieces, pieces, joins, chunks);
}

// Everything up to the row starts for n <= kSmallSort, one block.
constexpr int kSmallWarps = kSmallSort / kWarpItems;
constexpr int kSmallThreads = kSmallWarps * 32;
__global__ void __launch_bounds__(kSmallThreads)
small_sort_kernel(SortIn in, int n, int passes, int bits, uint32_t* __restrict__ pos_out,
                  uint32_t* __restrict__ start, uint32_t* __restrict__ n_pieces,
                  Piece* __restrict__ pieces, uint32_t* __restrict__ joins, int chunks) {
  extern __shared__ uint32_t sm[];
  uint32_t* keys = sm;
  uint32_t* pos = sm + kSmallSort;
  uint32_t* h = sm + 2 * kSmallSort;             // [kSmallWarps][bins]
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << bits;
  if (threadIdx.x == 0) *n_pieces = 0;
  const int w0 = warp * kWarpItems;
  uint32_t key[kWarpItems / 32], p[kWarpItems / 32];
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u) {
    const int i = w0 + u * 32 + lane;
    key[u] = i < n ? id_key(in, i) : 0xffffffffu;
    p[u] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int b = threadIdx.x; b < kSmallWarps * bins; b += kSmallThreads) h[b] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kWarpItems / 32; ++u)
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
    for (int u = 0; u < kWarpItems / 32; ++u) {
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
      for (int u = 0; u < kWarpItems / 32; ++u) {
        const int i = w0 + u * 32 + lane;
        if (i < n) key[u] = keys[i], p[u] = pos[i];
      }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSmallThreads) pos_out[i] = pos[i];
  for (int i0 = 0; i0 <= n; i0 += kSmallThreads)
    row_starts([&](uint32_t i) { return keys[i]; }, n, (uint32_t)in.n_v, i0 + threadIdx.x, start,
               n_pieces, pieces, joins, chunks);
}

struct SumArgs {
  const uint32_t *start, *pos, *n_pieces;
  const Piece* pieces;
  uint32_t* joins;
  const void* yb;
  void *wb, *part;
  double scale;
  int64_t n_v;
  int n_d, chunks, piece_blocks;
  bool add;
};

// The sum of one vector of columns over positions from .. from + len - 1, in order.
template <class T, int VEC>
__device__ __forceinline__ void sum_rows(const uint32_t* __restrict__ pos, uint32_t from,
                                         uint32_t len, const T* __restrict__ yb, int n_d, int col,
                                         acc_t<T> (&acc)[VEC]) {
  using V = Vec<T, VEC>;
  constexpr int U = 8;
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0;
  for (uint32_t i = 0; i < len; i += U) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < len)
        r[u] = *reinterpret_cast<const V*>(yb + (int64_t)pos[from + i + u] * n_d + col);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < len)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += load_acc<T>(r[u].v[k]);
  }
}

// VEC columns of a gradient row, in pieces of 16 bytes.
template <class A, int VEC>
__device__ __forceinline__ void put(A* p, const A (&v)[VEC], A scale, bool add) {
  constexpr int W = VEC * sizeof(A) >= 16 ? 16 / (int)sizeof(A) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += W) {
    Vec<A, W> o;
    if (add) o = *reinterpret_cast<const Vec<A, W>*>(p + i);
#pragma unroll
    for (int k = 0; k < W; ++k) o.v[k] = add ? o.v[k] + v[i + k] * scale : v[i + k] * scale;
    *reinterpret_cast<Vec<A, W>*>(p + i) = o;
  }
}

constexpr int kRowsPerWarp = 8;

// Blocks 0 .. piece_blocks - 1 take the pieces of long rows, the others eight
// table rows a warp, zeros included.
template <class T, int VEC>
__global__ void __launch_bounds__(kThreads)
row_sum_kernel(SumArgs p) {
  using A = acc_t<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* yb = (const T*)p.yb;
  A* wb = (A*)p.wb;
  const A scale = (A)p.scale;
  if ((int)blockIdx.x < p.piece_blocks) {
    __shared__ A sm[kWarps][32 * VEC];
    __shared__ bool last;
    const uint32_t items = *p.n_pieces * (uint32_t)p.chunks;
    for (uint32_t it = blockIdx.x; it < items; it += p.piece_blocks) {
      const Piece q = p.pieces[it / p.chunks];
      const int chunk = it % p.chunks, col = (chunk * 32 + lane) * VEC;
      const uint32_t sub = (q.len + kWarps - 1) / kWarps, i0 = min(q.len, warp * sub);
      A acc[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0;
      if (col < p.n_d)
        sum_rows<T, VEC>(p.pos, q.from + i0, min(sub, q.len - i0), yb, p.n_d, col, acc);
#pragma unroll
      for (int k = 0; k < VEC; ++k) sm[warp][k * 32 + lane] = acc[k];
      __syncthreads();
      A* part = (A*)p.part;
      if (warp == 0 && col < p.n_d) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          acc[k] = sm[0][k * 32 + lane];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) acc[k] += sm[w][k * 32 + lane];
        }
        if (q.count == 1)
          put<A, VEC>(wb + (int64_t)q.v * p.n_d + col, acc, scale, p.add);
        else
          put<A, VEC>(part + (int64_t)(it / p.chunks) * p.n_d + col, acc, A(1), false);
      }
      if (q.count > 1) {
        // the last block of this row and these columns adds the pieces in order
        if (warp == 0) {
          __threadfence();
          __syncwarp();
          if (lane == 0)
            last = atomicAdd(&p.joins[(int64_t)q.first * p.chunks + chunk], 1u) == q.count - 1;
        }
        __syncthreads();
        if (last && warp == 0 && col < p.n_d) {
          __threadfence();
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] = 0;
          constexpr int U = 4;
          for (uint32_t j = 0; j < q.count; j += U) {
            Vec<A, VEC> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (j + u < q.count)
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                  r[u].v[k] = __ldcg(part + (int64_t)(q.first + j + u) * p.n_d + col + k);
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (j + u < q.count)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] += r[u].v[k];
          }
          put<A, VEC>(wb + (int64_t)q.v * p.n_d + col, acc, scale, p.add);
        }
      }
      __syncthreads();
    }
    return;
  }
  const int64_t v0 =
      ((int64_t)(blockIdx.x - p.piece_blocks) * (kThreads / 32) + warp) * kRowsPerWarp;
  if (v0 >= p.n_v) return;
  const uint32_t bound = lane <= kRowsPerWarp && v0 + lane <= p.n_v ? p.start[v0 + lane] : 0u;
  const int rows = (int)min((int64_t)kRowsPerWarp, p.n_v - v0);
  for (int q = 0; q < rows; ++q) {
    const uint32_t i0 = __shfl_sync(0xffffffffu, bound, q);
    const uint32_t len = __shfl_sync(0xffffffffu, bound, q + 1) - i0;
    if (len > kShort || (p.add && len == 0)) continue;
    A* row = wb + (v0 + q) * p.n_d;
    for (int col = lane * VEC; col < p.n_d; col += 32 * VEC) {
      A acc[VEC];
      sum_rows<T, VEC>(p.pos, i0, len, yb, p.n_d, col, acc);
      put<A, VEC>(row + col, acc, scale, p.add);
    }
  }
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

// Columns a warp covers at once: a vector of VEC a lane.
template <class T, class F>
stade_status with_vec(int align_t, int align_p, F&& f) {
  using std::integral_constant;
  constexpr int W = 16 / (int)sizeof(T);
  if (align_t >= 16 && align_p >= 16) return f(integral_constant<int, W>{});
  if constexpr (sizeof(T) == 2)
    if (align_t >= 4 && align_p >= 8) return f(integral_constant<int, 2>{});
  return f(integral_constant<int, 1>{});
}
int64_t most_pieces(int64_t n_s) { return n_s / (kShort + 1) + n_s / kPiece + 1; }

struct Scratch {
  uint32_t *keys[2], *pos[2], *counts, *start, *n_pieces, *joins;
  Piece* pieces;
  char* part;
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
  take(&s.start, n_v + 1);
  take(&s.n_pieces, 1);
  take(&s.pieces, most_pieces(n_s));
  take(&s.joins, most_pieces(n_s) * ((n_d + 31) / 32));
  // partial sums: only of rows of more than kPiece positions
  if (n_s > kPiece) take(&s.part, (size_t)most_pieces(n_s) * n_d * 8);
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
    return with_vec<T>(row_align(n_d * sizeof(T), {w, y}), 16, [&](auto vec) {
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
      return with_vec<T>(row_align(n_d * sizeof(T), {yb}), row_align(n_d * sizeof(A), {wb}),
                         [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        const int chunks = (int)((n_d + 32 * VEC - 1) / (32 * VEC));
        const uint32_t* pos;
        if (n_s <= kSmallSort) {
          const size_t smem = (2 * kSmallSort + (size_t)kSmallWarps * bins) * 4;
          STADE_CUDA(cudaFuncSetAttribute(small_sort_kernel,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
          small_sort_kernel<<<1, kSmallThreads, smem, s>>>(
              SortIn{ids, nullptr, nullptr, base, n_v}, (int)n_s, p.passes, p.bits, sc.pos[0],
              sc.start, sc.n_pieces, sc.pieces, sc.joins, chunks);
          STADE_CHECK_LAUNCH();
          pos = sc.pos[0];
        } else {
          const int64_t per_pass = p.blocks << p.bits;
          for (int i = 0; i < p.passes; ++i) {
            const SortIn in{i == 0 ? ids : nullptr, sc.keys[(i + 1) & 1], sc.pos[(i + 1) & 1], base,
                            n_v};
            uint32_t* counts = sc.counts + i * per_pass;
            if (i == 0) {
              sort_count_kernel<<<(unsigned)p.blocks, kThreads, 0, s>>>(
                  in, n_s, bins, counts, (p.passes - 1) * per_pass, sc.n_pieces);
              STADE_CHECK_LAUNCH();
            }
            const bool scan = p.blocks > kFusedScan;
            if (scan) {
              scan_kernel<<<1, 1024, 0, s>>>(counts, per_pass);
              STADE_CHECK_LAUNCH();
            }
            sort_scatter_kernel<<<(unsigned)p.blocks, kThreads, 0, s>>>(
                in, n_s, i * p.bits, bins, counts, scan,
                i + 1 < p.passes ? counts + per_pass : nullptr, sc.keys[i & 1], sc.pos[i & 1]);
            STADE_CHECK_LAUNCH();
          }
          const int last = (p.passes - 1) & 1;
          row_start_kernel<<<ceil_div_u(n_s + 1, kThreads), kThreads, 0, s>>>(
              sc.keys[last], (uint32_t)n_s, (uint32_t)n_v, sc.start, sc.n_pieces, sc.pieces,
              sc.joins, chunks);
          STADE_CHECK_LAUNCH();
          pos = sc.pos[last];
        }
        SumArgs a{sc.start, pos, sc.n_pieces, sc.pieces, sc.joins, yb, wb, sc.part, scale, n_v,
                  (int)n_d, chunks, 0, add};
        // blocks for the pieces, where there can be any
        a.piece_blocks =
            n_s > kShort ? (int)std::min<int64_t>(148 * 4, most_pieces(n_s) * chunks) : 0;
        const int64_t row_blocks =
            (n_v + kRowsPerWarp * (kThreads / 32) - 1) / (kRowsPerWarp * (kThreads / 32));
        row_sum_kernel<T, VEC><<<(unsigned)(a.piece_blocks + row_blocks), kThreads, 0, s>>>(a);
        STADE_CHECK_LAUNCH();
        return (stade_status)STADE_OK;
      });
    });
    if (st != STADE_OK) return st;
  }
  if (consumes(opts)) STADE_CUDA(cudaMemsetAsync(yb, 0, (size_t)n_s * n_d * dtype_size(dtype), s));
  return STADE_OK;
}
