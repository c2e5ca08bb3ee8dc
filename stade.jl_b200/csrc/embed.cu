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

#include <initializer_list>

#include "token_ops.cuh"

namespace stade {
namespace {

__device__ int g_embed_error = 0;

constexpr int kThreads = 256;

template <class T>
__global__ void __launch_bounds__(kThreads)
embed_fwd_kernel(const T* __restrict__ w, const int64_t* __restrict__ ids, T* __restrict__ y,
                 acc_t<T> scale, int64_t base, int64_t n_v, int64_t n_d) {
  const int64_t s = blockIdx.x;
  const int64_t v = ids[s] - base;
  const bool ok = v >= 0 && v < n_v;
  if (v >= n_v && threadIdx.x == 0) g_embed_error = 1;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads)
    y[s * n_d + d] = round_to<T>(ok ? scale * load_acc<T>(w[v * n_d + d]) : acc_t<T>(0));
}

// ---- stable radix sort of (key, position) -------------------------------------
// key = v, or n_v for padding. A pass sorts by one digit of at most 9 bits:
// counts per block, one scan over [digit][block], and a scatter in which each
// warp walks its own stretch of the block's elements in order.
constexpr int kMaxBins = 512;
constexpr int kWarps = 8;
constexpr int kWarpItems = 256;
constexpr int kChunk = kWarps * kWarpItems;   // elements of one block

struct SortIn {
  const int64_t* ids;      // first pass: keys from the ids, positions 0 .. n - 1
  const uint32_t* keys;    // later passes
  const uint32_t* pos;
  int64_t base, n_v;
};
__device__ __forceinline__ uint32_t sort_key(const SortIn& in, int64_t i) {
  if (!in.ids) return in.keys[i];
  const int64_t v = in.ids[i] - in.base;
  if (v >= in.n_v) g_embed_error = 1;
  return (uint32_t)(v >= 0 && v < in.n_v ? v : in.n_v);
}

__global__ void __launch_bounds__(kThreads)
sort_count_kernel(SortIn in, int64_t n, int shift, int bins, uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[kMaxBins];
  for (int b = threadIdx.x; b < bins; b += kThreads) h[b] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kChunk, i1 = min(n, i0 + kChunk);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
    atomicAdd(&h[(sort_key(in, i) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads)
    counts[(int64_t)b * gridDim.x + blockIdx.x] = h[b];
}

// exclusive scan in place, one block
__global__ void __launch_bounds__(1024) scan_kernel(uint32_t* __restrict__ v, int64_t n) {
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (int64_t i0 = 0; i0 < n; i0 += 1024) {
    const int64_t i = i0 + threadIdx.x;
    const uint32_t x = i < n ? v[i] : 0;
    uint32_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      uint32_t t = sums[lane], a = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, a, o);
        if (lane >= o) a += u;
      }
      sums[lane] = a;
    }
    __syncthreads();
    const uint32_t before = carry + (warp ? sums[warp - 1] : 0u) + inc - x;
    if (i < n) v[i] = before;
    carry += sums[31];
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(SortIn in, int64_t n, int shift, int bins, const uint32_t* __restrict__ starts,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t h[kWarps][kMaxBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&h[0][0])[b] = 0;
  __syncthreads();
  const int64_t w0 = (int64_t)blockIdx.x * kChunk + warp * kWarpItems;
  uint32_t key[kWarpItems / 32];
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u) {
    const int64_t i = w0 + u * 32 + lane;
    key[u] = i < n ? sort_key(in, i) : 0xffffffffu;
  }
#pragma unroll
  for (int u = 0; u < kWarpItems / 32; ++u)
    if (w0 + u * 32 + lane < n) atomicAdd(&h[warp][(key[u] >> shift) & (bins - 1)], 1u);
  __syncthreads();
  // per digit: this block's start, then the warps one after the other
  for (int b = threadIdx.x; b < bins; b += kThreads) {
    uint32_t at = starts[(int64_t)b * gridDim.x + blockIdx.x];
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
    }
  }
}

// start[v] = number of sorted keys below v, v = 0 .. n_v
__global__ void __launch_bounds__(kThreads)
row_start_kernel(const uint32_t* __restrict__ keys, uint32_t n, int64_t n_v,
                 uint32_t* __restrict__ start) {
  const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (v > n_v) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  start[v] = lo;
}

template <class T>
__global__ void __launch_bounds__(kThreads)
row_sum_kernel(const uint32_t* __restrict__ start, const uint32_t* __restrict__ pos,
               const T* __restrict__ yb, acc_t<T>* __restrict__ wb, acc_t<T> scale, int64_t n_d,
               bool add) {
  const int64_t v = blockIdx.x;
  const uint32_t i0 = start[v], i1 = start[v + 1];
  if (add && i0 == i1) return;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) {
    acc_t<T> s = 0;
    for (uint32_t i = i0; i < i1; ++i) s += load_acc<T>(yb[(int64_t)pos[i] * n_d + d]);
    s *= scale;
    wb[v * n_d + d] = add ? wb[v * n_d + d] + s : s;
  }
}

struct SortPlan {
  int passes, bits;      // digits, bits of a digit
  int64_t blocks;
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

struct Scratch {
  uint32_t *keys[2], *pos[2], *counts, *start;
};
template <class S>
void layout(S& z, int64_t n_s, int64_t n_v, Scratch* out) {
  const SortPlan p = sort_plan(n_s, n_v);
  Scratch s{};
  auto take = [&](size_t n) {
    if constexpr (std::is_same<S, Sizer>::value) {
      z.template take<uint32_t>(n);
      return (uint32_t*)nullptr;
    } else {
      return z.template take<uint32_t>(n);
    }
  };
  for (int i = 0; i < 2; ++i) {
    s.keys[i] = take(n_s);
    s.pos[i] = take(n_s);
  }
  s.counts = take((size_t)p.blocks << p.bits);
  s.start = take(n_v + 1);
  if (out) *out = s;
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
    embed_fwd_kernel<T><<<(unsigned)n_s, kThreads, 0, s>>>((const T*)w, ids, (T*)y,
                                                           (acc_t<T>)scale, base, n_v, n_d);
    STADE_CHECK_LAUNCH();
    return (stade_status)STADE_OK;
  });
}

extern "C" size_t stade_embed_b_workspace(int64_t n_s, int64_t n_v, int64_t n_d) {
  if (n_s <= 0 || n_v <= 0 || n_d <= 0) return 0;
  Sizer z;
  layout(z, n_s, n_v, nullptr);
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
    Scratch sc;
    layout(c, n_s, n_v, &sc);
    const SortPlan p = sort_plan(n_s, n_v);
    const int bins = 1 << p.bits;
    for (int i = 0; i < p.passes; ++i) {
      const SortIn in{i == 0 ? ids : nullptr, sc.keys[(i + 1) & 1], sc.pos[(i + 1) & 1], base, n_v};
      sort_count_kernel<<<(unsigned)p.blocks, kThreads, 0, s>>>(in, n_s, i * p.bits, bins, sc.counts);
      STADE_CHECK_LAUNCH();
      scan_kernel<<<1, 1024, 0, s>>>(sc.counts, p.blocks << p.bits);
      STADE_CHECK_LAUNCH();
      sort_scatter_kernel<<<(unsigned)p.blocks, kThreads, 0, s>>>(
          in, n_s, i * p.bits, bins, sc.counts, sc.keys[i & 1], sc.pos[i & 1]);
      STADE_CHECK_LAUNCH();
    }
    const int last = (p.passes - 1) & 1;
    row_start_kernel<<<ceil_div_u(n_v + 1, kThreads), kThreads, 0, s>>>(
        sc.keys[last], (uint32_t)n_s, n_v, sc.start);
    STADE_CHECK_LAUNCH();
    st = with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      row_sum_kernel<T><<<(unsigned)n_v, kThreads, 0, s>>>(sc.start, sc.pos[last], (const T*)yb,
                                                           (acc_t<T>*)wb, (acc_t<T>)scale, n_d, add);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
    if (st != STADE_OK) return st;
  }
  if (consumes(opts)) STADE_CUDA(cudaMemsetAsync(yb, 0, (size_t)n_s * n_d * dtype_size(dtype), s));
  return STADE_OK;
}
