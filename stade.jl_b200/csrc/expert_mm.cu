// expert_mm and expert_mm_b: matrix products grouped by expert, with ragged
// groups whose bounds are on the device.
//
//   rows off[e] .. off[e + 1] - 1 belong to expert e (off has n_e + 1 entries)
//   y[s, :] = x[s, :] W[e]                    W: n_e x n_i x n_o
//   xb[s, :] += yb[s, :] W[e]^T
//   wb[e] += sum over the expert's rows of x[s, :]^T yb[s, :]
//
// Rows in no group get y = 0 and add nothing. The bounds are read on the
// device, so a router's counts never visit the host: one small kernel cuts
// every group into row tiles, and the product kernels walk that list. Bounds
// that fall or leave 0 .. n_s are clamped and set the device error word.
//
// The products run on the tensor cores (expert_tc.cu) for 16-bit arrays and
// Float32, on the CUDA cores for Float64, for 16-bit arrays of widths that are
// multiples of 8 but that do not start on 16-byte boundaries, and for Float32
// with a handful of rows a group. The second of these is slow: 4096 rows, 4
// experts, 2048 -> 4096 in bf16 3,129 us forward and 6,395 in reverse, 62 and 134
// on the boundary; widths of 2044 -> 4092, which are packed first, 102 and 183
// wherever they start. Float64, 2048 -> 1024: 1,079 and 2,164 us.

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "expert_tc.cuh"
#include "token_ops.cuh"

namespace stade {
namespace {

__device__ int g_expert_error = 0;

using Tile = ExpertTile;

constexpr int kTile = 64;       // rows and columns of a CUDA-core tile
constexpr int kStep = 16;

// Inclusive scan of one value per thread over a block of 1024; `sm`: 32 values.
template <class F>
__device__ __forceinline__ long long block_scan(long long v, long long* sm, F op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(u, v);
  }
  if (lane == 31) sm[warp] = v;
  __syncthreads();
  long long t = sm[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t = op(u, t);
  }
  const long long before = __shfl_sync(0xffffffffu, t, warp > 0 ? warp - 1 : 0);
  if (warp > 0) v = op(before, v);
  __syncthreads();
  return v;
}

// One block. bounds[0 .. n_e]: the clamped, rising bounds; tiles of at most
// `tile` rows of every group, then of the rows in no group; count[0]: how many.
__global__ void __launch_bounds__(1024)
plan_kernel(const int64_t* __restrict__ off, int64_t n_s, int64_t n_e, int tile,
            int64_t* __restrict__ bounds, Tile* __restrict__ tiles, int* __restrict__ count) {
  __shared__ long long sm[32];
  __shared__ long long edge[1024];
  __shared__ long long last;
  const int t = threadIdx.x;
  before_next();
  auto larger = [](long long a, long long b) { return a > b ? a : b; };
  auto sum = [](long long a, long long b) { return a + b; };
  long long low = 0, low_end = 0;     // the bound before this pass's first, the first of all
  int done = 0;                       // tiles so far
  // pass r: entries 1023 r .. 1023 r + 1023, the last of them the next pass's first
  for (int64_t e0 = 0; e0 <= n_e; e0 += 1023) {
    const int64_t e = e0 + t;
    long long v = 0;
    if (e <= n_e) {
      const long long raw = off[e];
      if (raw < 0 || raw > n_s || (e > 0 && raw < off[e - 1])) g_expert_error = 1;
      v = min(max(raw, 0ll), (long long)n_s);
    }
    // rising bounds: a running maximum of the clamped entries
    v = larger(block_scan(v, sm, larger), low);
    edge[t] = v;
    if (e <= n_e) bounds[e] = v;
    if (t == 1023) last = v;
    __syncthreads();
    low = last;
    if (e0 == 0) low_end = edge[0];
    const bool group = t < 1023 && e < n_e;
    const long long a = v, b = group ? edge[t + 1] : v;
    const long long mine = group ? (b - a + tile - 1) / tile : 0;
    const long long upto = block_scan(mine, sm, sum);
    int at = done + (int)(upto - mine);
    for (long long i = 0; i < mine; ++i, ++at)
      tiles[at] = Tile{(int)e, (int)(a + i * tile), (int)min((long long)tile, b - a - i * tile), 0};
    if (t == 1023) last = upto;
    __syncthreads();
    done += (int)last;
    __syncthreads();
  }
  // rows before the first bound and after the last
  const long long top = low;
  const long long head = (low_end + tile - 1) / tile, foot = (n_s - top + tile - 1) / tile;
  for (long long i = t; i < head + foot; i += 1024) {
    const long long a = i < head ? i * tile : top + (i - head) * tile;
    const long long z = i < head ? low_end : n_s;
    tiles[done + i] = Tile{-1, (int)a, (int)min((long long)tile, z - a), 0};
  }
  if (t == 0) count[0] = done + (int)(head + foot);
}

// C[m][n] (+)= sum_k A(m, k) B(k, n) of one 64 x 64 tile, A(m, k) =
// a[m am + k ak], B(k, n) = b[k bk + n bn], C[m][n] = c[m ldc + n].
template <class T, class O>
__device__ __forceinline__ void simt_tile(const T* __restrict__ a, int64_t am, int64_t ak,
                                          const T* __restrict__ b, int64_t bk, int64_t bn,
                                          O* __restrict__ c, int64_t ldc, int M, int N, int64_t K,
                                          bool add) {
  using A = acc_t<T>;
  __shared__ A as[kStep][kTile + 1], bs[kStep][kTile + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  A acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += kStep) {
    for (int i = tid; i < kStep * kTile; i += 256) {
      const int ka = ak == 1 ? i % kStep : i / kTile, ma = ak == 1 ? i / kStep : i % kTile;
      as[ka][ma] = ma < M && k0 + ka < K ? load_acc<T>(a[ma * am + (k0 + ka) * ak]) : A(0);
      const int kb = bk == 1 ? i % kStep : i / kTile, nb = bk == 1 ? i / kStep : i % kTile;
      bs[kb][nb] = nb < N && k0 + kb < K ? load_acc<T>(b[(k0 + kb) * bk + nb * bn]) : A(0);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      A ra[4], rb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ra[i] = as[k][ty + 16 * i], rb[i] = bs[k][tx + 16 * i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += ra[i] * rb[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = ty + 16 * i, n = tx + 16 * j;
      if (m < M && n < N) {
        O* p = c + m * ldc + n;
        *p = round_to<O>(add ? load_acc<O>(*p) + acc[i][j] : acc[i][j]);
      }
    }
}

// rows x width: y = x W (trans false) or xb = yb W^T (trans true)
template <class T>
__global__ void __launch_bounds__(256)
expert_rows_kernel(const T* __restrict__ in, const T* __restrict__ w, T* __restrict__ out,
                   const Tile* __restrict__ tiles, const int* __restrict__ count, int64_t n_i,
                   int64_t n_o, bool trans, bool add) {
  if ((int)blockIdx.x >= *count) return;
  const Tile t = tiles[blockIdx.x];
  const int64_t width = trans ? n_i : n_o, depth = trans ? n_o : n_i;
  const int64_t n0 = (int64_t)blockIdx.y * kTile;
  const T* wt = w + (int64_t)max(t.expert, 0) * n_i * n_o + (trans ? n0 * n_o : n0);
  simt_tile<T, T>(in + (int64_t)t.row * depth, depth, 1, wt, trans ? 1 : n_o, trans ? n_o : 1,
                  out + (int64_t)t.row * width + n0, width, t.rows,
                  (int)min((int64_t)kTile, width - n0), t.expert < 0 ? 0 : depth, add);
}

template <class T>
__global__ void __launch_bounds__(256)
expert_wgrad_kernel(const T* __restrict__ x, const T* __restrict__ yb, acc_t<T>* __restrict__ wb,
                    const int64_t* __restrict__ bounds, int64_t n_i, int64_t n_o, bool add) {
  const int64_t e = blockIdx.z, i0 = (int64_t)blockIdx.y * kTile, o0 = (int64_t)blockIdx.x * kTile;
  const int64_t a = bounds[e], b = bounds[e + 1];
  simt_tile<T, acc_t<T>>(x + a * n_i + i0, 1, n_i, yb + a * n_o + o0, n_o, 1,
                         wb + (e * n_i + i0) * n_o + o0, n_o, (int)min((int64_t)kTile, n_i - i0),
                         (int)min((int64_t)kTile, n_o - o0), b - a, add);
}

// ---- few rows, Float32 ------------------------------------------------------------
// With a handful of rows a group the time is one read of the weights. The
// tensor cores' path writes them out as three planes first and reads those: six
// times the bytes (6 rows, 2 experts, 2328 -> 3688: 107 us, of which 10 us is
// the read). Here tiles of kFew rows multiply on the CUDA cores, the rows in
// shared memory, the weights read once per tile straight into registers: once in
// all when no group has more than kFew rows.
//
// The bounds are on the device, so the path goes by the average. Measured with
// eight rows a group, spread evenly and all in one group (whose weights are then
// read once per eight rows, and whose gradient few warps add up), against the
// tensor cores' path; y, xb, wb in us:
//   512 rows, 512 x 512     even 30, 92, 30    69, 71, 55     one 30, 92, 74     59, 58, 48
//   4096 rows, 64 x 64      even 14, 90, 14    36, 36, 67     one 23, 99, 481    19, 20, 180
//   32768 rows, 64 x 64     even 59, 704, 69   219, 220, 463  one 126, 739, 5220 64, 64, 1364
constexpr int kFew = 8;
constexpr int kFewK = 512;      // depth of one block's share of y = x W
constexpr int kFewWarps = 8;

// y = x W: a block takes 32 V columns of a tile and kFewK of the depth, a warp
// an eighth of that; the warps' sums are added in order. part: [slice][row][n_o]
// where the depth takes several blocks, else y itself.
template <int V>
__global__ void __launch_bounds__(32 * kFewWarps)
few_forward_kernel(const float* __restrict__ x, const float* __restrict__ w,
                   float* __restrict__ part, const Tile* __restrict__ tiles,
                   const int* __restrict__ count, int n_i, int n_o, int64_t n_s) {
  __shared__ __align__(16) float xs[kFewK][kFew];
  __shared__ float red[kFewWarps][kFew][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  after_previous();
  if ((int)blockIdx.x >= *count) return;
  const Tile t = tiles[blockIdx.x];
  const int k0 = blockIdx.z * kFewK, depth = t.expert < 0 ? 0 : min(kFewK, n_i - k0);
  const int o = (blockIdx.y * 32 + lane) * V;
  for (int i = threadIdx.x; i < kFew * depth; i += 32 * kFewWarps) {
    const int r = i / depth, k = i - r * depth;
    xs[k][r] = r < t.rows ? x[(int64_t)(t.row + r) * n_i + k0 + k] : 0.f;
  }
  __syncthreads();
  float acc[kFew][V] = {};
  if (o < n_o) {
    const float* wp = w + ((int64_t)max(t.expert, 0) * n_i + k0) * n_o + o;
    const int per = (depth + kFewWarps - 1) / kFewWarps, a = warp * per, z = min(depth, a + per);
    constexpr int U = 8;
    for (int k = a; k < z; k += U) {
      Vec<float, V> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u < z) r[u] = *reinterpret_cast<const Vec<float, V>*>(wp + (int64_t)(k + u) * n_o);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u < z)
#pragma unroll
          for (int q = 0; q < kFew; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[q][v] = fmaf(xs[k + u][q], r[u].v[v], acc[q][v]);
    }
  }
#pragma unroll
  for (int q = 0; q < kFew; ++q)
#pragma unroll
    for (int v = 0; v < V; ++v) red[warp][q][v * 32 + lane] = acc[q][v];
  __syncthreads();
  // warp q adds up row q
  if (warp < t.rows && o < n_o) {
    float* out = part + ((int64_t)blockIdx.z * n_s + t.row + warp) * n_o + o;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kFewWarps; ++j) s += red[j][warp][v * 32 + lane];
      out[v] = s;
    }
  }
}
// y = the slices' sums, in order
__global__ void __launch_bounds__(256)
few_join_kernel(const float* __restrict__ part, float* __restrict__ y, int64_t n, int slices) {
  after_previous();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) y[i] = ordered_sum(part + i, slices, n);
}

// xb (+)= yb W^T: a block takes eight rows of W, its warps every eighth stretch
// of 32 V columns; the 64 sums of a warp are halved down to two a lane, and the
// warps' added in order.
template <int V>
__global__ void __launch_bounds__(32 * kFewWarps)
few_input_kernel(const float* __restrict__ yb, const float* __restrict__ w, float* __restrict__ xb,
                 const Tile* __restrict__ tiles, const int* __restrict__ count, int n_i, int n_o,
                 bool add) {
  constexpr int kRows = 8;
  __shared__ float red[kFewWarps][kRows * kFew];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  after_previous();
  if ((int)blockIdx.x >= *count) return;
  const Tile t = tiles[blockIdx.x];
  const int i0 = blockIdx.y * kRows;
  float acc[kRows * kFew] = {};            // [row of W][row of the tile]
  const float* wp = w + ((int64_t)max(t.expert, 0) * n_i + i0) * n_o;
  const float* yp = yb + (int64_t)t.row * n_o;
  for (int c = (warp * 32 + lane) * V; c < (t.expert < 0 ? 0 : n_o); c += kFewWarps * 32 * V) {
    Vec<float, V> r[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (i0 + j < n_i) r[j] = *reinterpret_cast<const Vec<float, V>*>(wp + (int64_t)j * n_o + c);
#pragma unroll
    for (int q = 0; q < kFew; ++q)
      if (q < t.rows) {
        const Vec<float, V> g = *reinterpret_cast<const Vec<float, V>*>(yp + (int64_t)q * n_o + c);
#pragma unroll
        for (int j = 0; j < kRows; ++j)
          if (i0 + j < n_i)
#pragma unroll
            for (int v = 0; v < V; ++v)
              acc[j * kFew + q] = fmaf(g.v[v], r[j].v[v], acc[j * kFew + q]);
      }
  }
#pragma unroll
  for (int n = 32; n > 1; n >>= 1) {
    const bool up = lane & (n / 2);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? acc[i] : acc[i + n], keep = up ? acc[i + n] : acc[i];
      acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, n / 2);
    }
  }
  red[warp][2 * lane] = acc[0];        // lane l has sums 2 l and 2 l + 1
  red[warp][2 * lane + 1] = acc[1];
  __syncthreads();
  const int i = i0 + (int)threadIdx.x / kFew, q = threadIdx.x % kFew;
  if (threadIdx.x < kRows * kFew && i < n_i && q < t.rows) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kFewWarps; ++j) s += red[j][threadIdx.x];
    float* o = xb + (int64_t)(t.row + q) * n_i + i;
    *o = add ? *o + s : s;
  }
}

// wb[e] (+)= sum over the group's rows of x^T yb: one write of the gradient. A
// warp takes four rows and 32 V columns of it and walks the group's rows. A
// group can hold all rows: after kFewChain of them the sums go to the gradient
// and begin anew, so that the error grows with the root of a chain's length and
// of their number, not of the rows'. (Kept in a second set of registers they cost
// a quarter of the time of groups of eight rows: 1,024 experts of 512 x 512, 441
// us so, 582.)
constexpr int kFewChain = 64;
template <int V>
__global__ void __launch_bounds__(32 * kFewWarps)
few_weight_kernel(const float* __restrict__ x, const float* __restrict__ yb, float* __restrict__ wb,
                  const int64_t* __restrict__ bounds, int n_i, int n_o, bool add) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  after_previous();
  const int64_t e = blockIdx.z, a = bounds[e], z = bounds[e + 1];
  const int i0 = (blockIdx.y * kFewWarps + warp) * 4, o = (blockIdx.x * 32 + lane) * V;
  if (i0 >= n_i || o >= n_o || (add && a == z)) return;
  int64_t s = a;
  do {
    const int64_t upto = min(z, s + kFewChain);
    float acc[4][V] = {};
    for (; s < upto; s += 4) {
      Vec<float, V> g[4];
      float f[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool in = s + u < upto;
        if (in) g[u] = *reinterpret_cast<const Vec<float, V>*>(yb + (s + u) * n_o + o);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[u][j] = in && i0 + j < n_i ? x[(s + u) * n_i + i0 + j] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (s + u < upto)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[j][v] = fmaf(f[u][j], g[u].v[v], acc[j][v]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < n_i) {
        float* p = wb + (e * n_i + i0 + j) * n_o + o;
        Vec<float, V> r;
        if (add) r = *reinterpret_cast<const Vec<float, V>*>(p);
#pragma unroll
        for (int v = 0; v < V; ++v) r.v[v] = add ? r.v[v] + acc[j][v] : acc[j][v];
        *reinterpret_cast<Vec<float, V>*>(p) = r;
      }
    add = true;
  } while (s < z);
}

// Whether the rows are few enough: no more than kFew a group on average.
bool few_rows(int dtype, int64_t n_s, int64_t n_e, int64_t n_i, int64_t n_o) {
  return dtype == STADE_F32 && n_s <= kFew * n_e && std::max(n_i, n_o) < (int64_t(1) << 18);
}
int64_t few_slices(int64_t n_i) { return (n_i + kFewK - 1) / kFewK; }

int64_t max_tiles(int64_t n_s, int64_t n_e, int tile) { return n_s / tile + n_e + 2; }

// Which path a call takes. The tensor cores read 16-bit operands whose rows
// start on 16-byte boundaries: arrays of a 16-bit type with widths that are
// multiples of 8 as they stand, other widths and Float32 from planes that
// expert_pack writes into the workspace. Float64, and 16-bit arrays that do
// not start on such a boundary, go to the CUDA cores.
bool packs(int dtype, int64_t n_i, int64_t n_o) {
  return dtype == STADE_F32 || n_i % 8 || n_o % 8;
}
bool on_tensor_cores(int dtype, int64_t n_i, int64_t n_o, std::initializer_list<const void*> ptrs) {
  if (dtype == STADE_F64) return false;
  return packs(dtype, n_i, n_o) || row_align(16, ptrs) == 16;
}
int64_t pitch8(int64_t n) { return (n + 7) / 8 * 8; }

struct Plan {
  int64_t* bounds;
  Tile* tiles;
  int* count;
  uint16_t *x, *w, *yb;      // packed planes, where needed
  float* part;               // few rows: the depth slices' sums
};
// S: Sizer or Carver
template <class S>
Plan layout(S& z, int dtype, int64_t n_s, int64_t n_e, int64_t n_i, int64_t n_o, bool reverse) {
  Plan p{};
  auto take = [&](auto** to, size_t n) {
    using E = std::remove_pointer_t<std::remove_pointer_t<decltype(to)>>;
    if constexpr (std::is_same<S, Sizer>::value) z.template take<E>(n);
    else *to = z.template take<E>(n);
  };
  take(&p.bounds, n_e + 1);
  const bool few = few_rows(dtype, n_s, n_e, n_i, n_o);
  take(&p.tiles, max_tiles(n_s, n_e, few ? kFew : kTile));
  take(&p.count, 1);
  if (few && !reverse && few_slices(n_i) > 1) take(&p.part, few_slices(n_i) * n_s * n_o);
  if (!few && dtype != STADE_F64 && packs(dtype, n_i, n_o)) {
    const int64_t np = expert_planes(dtype);
    take(&p.x, np * n_s * pitch8(n_i));
    take(&p.w, np * n_e * n_i * pitch8(n_o));
    if (reverse) take(&p.yb, np * n_s * pitch8(n_o));
  }
  return p;
}
size_t plan_bytes(int dtype, int64_t n_s, int64_t n_e, int64_t n_i, int64_t n_o, bool reverse) {
  if (n_s <= 0 || n_e < 0 || n_i < 0 || n_o < 0) return 0;
  Sizer z;
  layout(z, dtype, n_s, n_e, n_i, n_o, reverse);
  return z.bytes();
}
stade_status make_plan(const Plan& p, const int64_t* off, int64_t n_s, int64_t n_e, int tile,
                       cudaStream_t s) {
  plan_kernel<<<1, 1024, 0, s>>>(off, n_s, n_e, tile, p.bounds, p.tiles, p.count);
  STADE_CHECK_LAUNCH();
  return STADE_OK;
}

// An operand for the tensor cores: d2 x d1 rows of d0 values, packed into
// `planes` first where the call packs.
stade_status operand(int dtype, const void* a, uint16_t* planes, int64_t d0, int64_t d1, int64_t d2,
                     ExpertOperand* out, cudaStream_t s) {
  if (!planes) {
    *out = ExpertOperand{a, d0, d1, d2, d0};
    return STADE_OK;
  }
  *out = ExpertOperand{planes, d0, d1, d2 * expert_planes(dtype), pitch8(d0)};
  return expert_pack(dtype, a, planes, d1 * d2, d0, pitch8(d0), s);
}

stade_status check_sizes(const char* who, int dtype, int64_t n_s, int64_t n_e, int64_t n_i,
                         int64_t n_o) {
  STADE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  STADE_REQUIRE(n_s >= 0 && n_e >= 0 && n_i >= 0 && n_o >= 0, "%s: negative size", who);
  int64_t t;
  STADE_REQUIRE(n_s < (int64_t(1) << 30) && n_e < (int64_t(1) << 16) - 2 &&
                    n_i < (int64_t(1) << 21) && n_o < (int64_t(1) << 21) &&
                    mul_ok(n_s, n_i + n_o, &t) && mul_ok(n_e, n_i * n_o, &t),
                "%s: size overflow", who);
  return STADE_OK;
}

}  // namespace

int expert_take_error() {
  int host = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&host, g_expert_error, sizeof(int)) != cudaSuccess) return -1;
  if (host) cudaMemcpyToSymbol(g_expert_error, &zero, sizeof(int));
  const int tc = expert_tc_take_error();
  return tc < 0 ? -1 : host | tc;
}

}  // namespace stade

using namespace stade;

extern "C" size_t stade_expert_mm_workspace(int dtype, int64_t n_s, int64_t n_e, int64_t n_i,
                                            int64_t n_o) {
  return plan_bytes(dtype, n_s, n_e, n_i, n_o, false);
}

extern "C" stade_status stade_expert_mm(int dtype, const void* x, const void* w, void* y,
                                        const int64_t* off, int64_t n_s, int64_t n_e, int64_t n_i,
                                        int64_t n_o, const stade_opts* opts) {
  stade_status st = check_sizes("expert_mm", dtype, n_s, n_e, n_i, n_o);
  if (st != STADE_OK) return st;
  if (n_s == 0 || n_o == 0) return STADE_OK;
  cudaStream_t s = stream_of(opts);
  STADE_REQUIRE(y, "expert_mm: null array argument");
  if (n_i == 0 || n_e == 0) {   // empty sums
    STADE_CUDA(cudaMemsetAsync(y, 0, (size_t)n_s * n_o * dtype_size(dtype), s));
    return STADE_OK;
  }
  STADE_REQUIRE(x && w && off, "expert_mm: null array argument");
  void* ws = nullptr;
  st = get_workspace(opts, stade_expert_mm_workspace(dtype, n_s, n_e, n_i, n_o), &ws);
  if (st != STADE_OK) return st;
  PhaseScope ph("expert_mm", s);
  Carver c(ws);
  const Plan p = layout(c, dtype, n_s, n_e, n_i, n_o, false);
  const bool few = few_rows(dtype, n_s, n_e, n_i, n_o);
  const bool tc = !few && on_tensor_cores(dtype, n_i, n_o, {x, w});
  st = make_plan(p, off, n_s, n_e, few ? kFew : tc ? kExpertTcRows : kTile, s);
  if (st != STADE_OK) return st;
  if (few) {
    const bool vec = row_align(n_o * 4, {w}) == 16;
    const int slices = (int)few_slices(n_i);
    const dim3 grid((unsigned)max_tiles(n_s, n_e, kFew), ceil_div_u(n_o, vec ? 128 : 32), slices);
    st = launch_next(vec ? few_forward_kernel<4> : few_forward_kernel<1>, grid, 32 * kFewWarps, 0,
                     s, (const float*)x, (const float*)w, slices > 1 ? p.part : (float*)y, p.tiles,
                     p.count, (int)n_i, (int)n_o, n_s);
    if (st != STADE_OK || slices == 1) return st;
    return launch_next(few_join_kernel, ceil_div_u(n_s * n_o, 256), 256, 0, s, p.part, (float*)y,
                       n_s * n_o, slices);
  }
  if (tc) {
    ExpertOperand xo, wo;
    st = operand(dtype, x, p.x, n_i, n_s, 1, &xo, s);
    if (st == STADE_OK) st = operand(dtype, w, p.w, n_o, n_i, n_e, &wo, s);
    if (st != STADE_OK) return st;
    return expert_tc_rows(dtype, xo, wo, y, p.tiles, p.count, max_tiles(n_s, n_e, kExpertTcRows),
                          n_i, n_o, false, false, s);
  }
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)max_tiles(n_s, n_e, kTile), ceil_div_u(n_o, kTile));
    expert_rows_kernel<T><<<grid, 256, 0, s>>>((const T*)x, (const T*)w, (T*)y, p.tiles, p.count,
                                               n_i, n_o, false, false);
    STADE_CHECK_LAUNCH();
    return (stade_status)STADE_OK;
  });
}

extern "C" size_t stade_expert_mm_b_workspace(int dtype, int64_t n_s, int64_t n_e, int64_t n_i,
                                              int64_t n_o) {
  return plan_bytes(dtype, n_s, n_e, n_i, n_o, true);
}

extern "C" stade_status stade_expert_mm_b(int dtype, const void* x, void* xb, const void* w,
                                          void* wb, void* yb, const int64_t* off, int64_t n_s,
                                          int64_t n_e, int64_t n_i, int64_t n_o,
                                          const stade_opts* opts) {
  stade_status st = check_sizes("expert_mm_b", dtype, n_s, n_e, n_i, n_o);
  if (st != STADE_OK) return st;
  cudaStream_t s = stream_of(opts);
  const bool add = accumulates(opts);
  const size_t wsize = dtype == STADE_F64 ? 8 : 4;
  if (n_s == 0 || n_e == 0 || n_i == 0 || n_o == 0) {   // empty sums
    if (!add && wb && n_e * n_i * n_o > 0)
      STADE_CUDA(cudaMemsetAsync(wb, 0, (size_t)(n_e * n_i * n_o) * wsize, s));
    if (!add && xb && n_s * n_i > 0)
      STADE_CUDA(cudaMemsetAsync(xb, 0, (size_t)(n_s * n_i) * dtype_size(dtype), s));
    if (consumes(opts) && yb && n_s * n_o > 0)
      STADE_CUDA(cudaMemsetAsync(yb, 0, (size_t)(n_s * n_o) * dtype_size(dtype), s));
    return STADE_OK;
  }
  STADE_REQUIRE(yb && off && (!xb || w) && (!wb || x), "expert_mm_b: null array argument");
  void* ws = nullptr;
  st = get_workspace(opts, stade_expert_mm_b_workspace(dtype, n_s, n_e, n_i, n_o), &ws);
  if (st != STADE_OK) return st;
  PhaseScope ph("expert_mm_b", s);
  Carver c(ws);
  const Plan p = layout(c, dtype, n_s, n_e, n_i, n_o, true);
  const bool few = few_rows(dtype, n_s, n_e, n_i, n_o);
  const bool tc = !few && on_tensor_cores(dtype, n_i, n_o, {wb ? x : yb, xb ? w : yb, yb});
  st = make_plan(p, off, n_s, n_e, few ? kFew : tc ? kExpertTcRows : kTile, s);
  if (st != STADE_OK) return st;
  if (few) {
    if (xb) {
      const bool vec = row_align(n_o * 4, {w, yb}) == 16;
      const dim3 grid((unsigned)max_tiles(n_s, n_e, kFew), ceil_div_u(n_i, 8));
      st = launch_next(vec ? few_input_kernel<4> : few_input_kernel<1>, grid, 32 * kFewWarps, 0, s,
                       (const float*)yb, (const float*)w, (float*)xb, p.tiles, p.count, (int)n_i,
                       (int)n_o, add);
    }
    if (st == STADE_OK && wb) {
      const bool vec = row_align(n_o * 4, {yb, wb}) == 16;
      const dim3 grid(ceil_div_u(n_o, vec ? 128 : 32), ceil_div_u(n_i, 4 * kFewWarps),
                      (unsigned)n_e);
      st = launch_next(vec ? few_weight_kernel<4> : few_weight_kernel<1>, grid, 32 * kFewWarps, 0,
                       s, (const float*)x, (const float*)yb, (float*)wb, p.bounds, (int)n_i,
                       (int)n_o, add);
    }
  } else if (tc) {
    ExpertOperand xo, wo, yo;
    st = operand(dtype, yb, p.yb, n_o, n_s, 1, &yo, s);
    if (st == STADE_OK && xb) {
      st = operand(dtype, w, p.w, n_o, n_i, n_e, &wo, s);
      if (st == STADE_OK)
        st = expert_tc_rows(dtype, yo, wo, xb, p.tiles, p.count,
                            max_tiles(n_s, n_e, kExpertTcRows), n_i, n_o, true, add, s);
    }
    if (st == STADE_OK && wb) {
      st = operand(dtype, x, p.x, n_i, n_s, 1, &xo, s);
      if (st == STADE_OK)
        st = expert_tc_wgrad(dtype, xo, yo, (float*)wb, p.bounds, n_e, n_i, n_o, add, s);
    }
  } else
    st = with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (xb) {
      const dim3 grid((unsigned)max_tiles(n_s, n_e, kTile), ceil_div_u(n_i, kTile));
      expert_rows_kernel<T><<<grid, 256, 0, s>>>((const T*)yb, (const T*)w, (T*)xb, p.tiles,
                                                 p.count, n_i, n_o, true, add);
      STADE_CHECK_LAUNCH();
    }
    if (wb) {
      const dim3 grid(ceil_div_u(n_o, kTile), ceil_div_u(n_i, kTile), (unsigned)n_e);
      expert_wgrad_kernel<T><<<grid, 256, 0, s>>>((const T*)x, (const T*)yb, (acc_t<T>*)wb,
                                                  p.bounds, n_i, n_o, add);
      STADE_CHECK_LAUNCH();
    }
    return (stade_status)STADE_OK;
  });
  if (st != STADE_OK) return st;
  if (consumes(opts))
    STADE_CUDA(cudaMemsetAsync(yb, 0, (size_t)n_s * n_o * dtype_size(dtype), s));
  return STADE_OK;
}
