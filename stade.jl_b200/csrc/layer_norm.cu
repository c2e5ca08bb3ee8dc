// layer_norm and layer_norm_b: normalisation over the last dimension and its
// reverse sweep with the sums over rows for the weight and the bias.
//
//   mean = sum_d x / n_d,  rstd = 1 / sqrt(sum_d (x - mean)^2 / n_d + eps)
//   h = (x - mean) rstd,   y = h w + b
//   g = yb w;  xb += rstd (g - mean(g) - h mean(g h))
//   wb += sum_s yb h,      bb += sum_s yb
//
// The forward leaves mean and rstd of every row on the tape (m_stack,
// r_stack); the reverse sweep reads them and x. The variance is summed from
// the centred values in a second pass, so a mean far from zero costs nothing
// but its own rounding.

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "tcgen05.cuh"
#include "token_ops.cuh"

namespace stade {
namespace {

// ---- rows held in registers -----------------------------------------------------
// Both sweeps are bound by memory: x in and y out, or x and yb in and xb out,
// each once. A row lives in registers, so nothing is read twice:
//  - rows of less than 1,536 bytes: a warp each, several rows in flight, w, b
//    and the sums over rows in the lanes' registers for all of a warp's rows;
//  - longer rows of arrays that start on 16-byte boundaries: the ring kernels,
//    a block each, the rows to come copied by cp.async.bulk into a ring in
//    shared memory, several rows ahead of the arithmetic;
//  - other rows: a group of G threads each, NV values a thread, read directly;
//  - rows too long for registers: read again from the caches. In reverse these
//    are rows past 24 KB, in two kernels of one value an access (4096 x 8192
//    Float32: 157 us, 61 by memory); clearing the seed in the second one's loop
//    keeps a thread to one row in flight (1,113 us with the default flags, 102
//    for the bytes that then move).

// Sums of two values over the block, the same in every thread. `red`: 2 x 2 x 32
// values, used alternately (`turn`), so that one barrier per sum is enough.
template <class A>
__device__ __forceinline__ void block_sum2(A& a, A& b, A (*red)[2][32], int turn, int warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  a = warp_sum(a);
  b = warp_sum(b);
  if (lane == 0) {
    red[turn][0][warp] = a;
    red[turn][1][warp] = b;
  }
  __syncthreads();
  a = warp_sum(lane < warps ? red[turn][0][lane] : A(0));
  b = warp_sum(lane < warps ? red[turn][1][lane] : A(0));
}
template <class T, int G, int NV>
__global__ void __launch_bounds__(G)
ln_fwd_kernel(const T* __restrict__ x, const acc_t<T>* __restrict__ w,
              const acc_t<T>* __restrict__ b, T* __restrict__ y, acc_t<T>* __restrict__ m_stack,
              acc_t<T>* __restrict__ r_stack, double eps, int n_d) {
  using A = acc_t<T>;
  __shared__ A red[2][2][32];
  const int t = threadIdx.x;
  const int64_t s = blockIdx.x;
  const T* xr = x + s * n_d;
  A c[NV], sum = 0, zero = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) c[i] = i * G + t < n_d ? load_acc<T>(xr[i * G + t]) : A(0);
#pragma unroll
  for (int i = 0; i < NV; ++i) sum += c[i];
  block_sum2(sum, zero, red, 0, G / 32);
  const A mean = sum / (A)n_d;
  A sq = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    c[i] -= mean;
    if (i * G + t < n_d) sq += c[i] * c[i];
  }
  block_sum2(sq, zero, red, 1, G / 32);
  const A rstd = A(1) / sqrt(sq / (A)n_d + (A)eps);
  if (t == 0) {
    m_stack[s] = mean;
    r_stack[s] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = i * G + t;
    if (d < n_d) y[s * n_d + d] = round_to<T>(c[i] * rstd * (w ? w[d] : A(1)) + (b ? b[d] : A(0)));
  }
}

// The reverse sweeps: blocks walk the rows at a stride of the grid, a thread
// keeps its columns of w and of the two sums over rows in registers. Per block
// one partial of each sum, added up in block order by ln_finish_kernel.
struct BwdArgs {
  const void *x, *w, *m, *r;
  void *xb, *yb, *part;
  int64_t n_s;
  int n_d;
  bool add, zero, sums;
};

template <class T, int G, int NV>
__global__ void __launch_bounds__(G)
ln_bwd_kernel(BwdArgs p) {
  using A = acc_t<T>;
  __shared__ A red[2][2][32];
  const int t = threadIdx.x;
  const T* x = (const T*)p.x;
  T* yb = (T*)p.yb;
  T* xb = (T*)p.xb;
  A w[NV], sw[NV], sb[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    w[i] = p.w && i * G + t < p.n_d ? ((const A*)p.w)[i * G + t] : A(1);
    sw[i] = sb[i] = A(0);
  }
  T nx[NV], ny[NV];       // the next row, loaded a row ahead
  A nm = 0, nr = 0;
  auto fetch = [&](int64_t q) {
    if (q >= p.n_s) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * G + t < p.n_d) {
        nx[i] = x[q * p.n_d + i * G + t];
        ny[i] = yb[q * p.n_d + i * G + t];
      }
    nm = ((const A*)p.m)[q];
    nr = ((const A*)p.r)[q];
  };
  fetch(blockIdx.x);
  int turn = 0;
  for (int64_t s = blockIdx.x; s < p.n_s; s += gridDim.x) {
    A h[NV], v[NV], sg = 0, sgh = 0;
    const A rstd = nr;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * G + t < p.n_d) {
        h[i] = (load_acc<T>(nx[i]) - nm) * rstd;
        v[i] = load_acc<T>(ny[i]);
      }
    fetch(s + gridDim.x);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * G + t < p.n_d) {
        const A g = v[i] * w[i];
        sg += g;
        sgh += g * h[i];
        sw[i] += v[i] * h[i];
        sb[i] += v[i];
      }
    block_sum2(sg, sgh, red, turn, G / 32);
    turn ^= 1;
    const A mg = sg / (A)p.n_d, mgh = sgh / (A)p.n_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = s * p.n_d + i * G + t;
      if (i * G + t < p.n_d) {
        if (xb) {
          const A o = rstd * (v[i] * w[i] - mg - h[i] * mgh);
          xb[at] = round_to<T>(p.add ? load_acc<T>(xb[at]) + o : o);
        }
        if (p.zero) yb[at] = round_to<T>(A(0));
      }
    }
  }
  if (!p.sums) return;
  A* part = (A*)p.part + (int64_t)blockIdx.x * 2 * p.n_d;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * G + t < p.n_d) {
      part[i * G + t] = sw[i];
      part[p.n_d + i * G + t] = sb[i];
    }
}

// ---- rings of rows -------------------------------------------------------------------
__device__ int g_norm_error = 0;

constexpr int kMaxStages = 8;

// Sums of N values over a warp by halving: each step adds one half of the values
// to the lanes that keep it. v[0] of lane l is then the sum of value l / (32 /
// N).
template <int N, class A>
__device__ __forceinline__ void halve(A (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int n = N, off = 16;
#pragma unroll
  for (int step = 0; step < 5; ++step, off >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = lane & off;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n) {
          const A send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
}
// v[i] = f(sum of v[i] over the warp), the same in every lane.
template <int N, class A, class F>
__device__ __forceinline__ void warp_sums(A (&v)[N], F f) {
  halve<N>(v);
  const A s = f(v[0]);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * (32 / N));
}

// v[i] = f(sum of v[i] over the block), the same in every thread: within a warp
// by halving, then one barrier and the warps' sums; f runs once, on the lanes that
// hold the sums, before they are spread (a division and a root per row in
// every thread were a third of the forward's instructions). `red`: 2 x 8 x 32
// values, zero where the block has no warp, used alternately (`turn`), so that
// no second barrier is needed.
template <int N, class A, class F>
__device__ __forceinline__ void block_sums(A (&v)[N], A (*red)[8][32], int turn, F f) {
  constexpr int kLanes = 32 / N;       // lanes per value
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  halve<N>(v);
  if (lane % kLanes == 0) red[turn][lane / kLanes][warp] = v[0];
  __syncthreads();
  A s = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) s += red[turn][lane / kLanes][lane % kLanes + i * kLanes];
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  s = f(s);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * kLanes);
}

// A stage holds R consecutive rows of up to two arrays, each copied as one
// piece. Copies start and end on 16-byte boundaries: where row bytes are no
// multiple of 16 a piece is widened to them (its rows then begin `mis` bytes
// into the stage), and what would pass the array's end, under 16 bytes, is
// copied by patch(). All of a block's threads call wait(); behind a barrier
// that follows their last read of a stage, thread 0 calls issue() for the rows
// that reuse it. A wait that runs out sets the error word and the block goes
// on without waiting, so that its barriers still match.
template <class T, int ARRAYS, bool WIDE>
struct Ring {
  const uint8_t* src[2];
  uint8_t* data;
  uint32_t bar0;
  int stages, R;
  uint32_t row_bytes, array_bytes;
  int64_t total;
  bool dead;
  __device__ __forceinline__ Ring(uint8_t* smem, int stages_, int rows, int n_d, int64_t n_s,
                                  const void* a, const void* b)
      : data(smem + 128), bar0(tc5::smem_u32(smem)), stages(stages_), R(rows),
        row_bytes(n_d * (uint32_t)sizeof(T)),
        array_bytes(WIDE ? rows * row_bytes : (rows * row_bytes + 31) & ~15u),
        total(n_s * row_bytes), dead(false) {
    src[0] = (const uint8_t*)a;
    src[1] = (const uint8_t*)b;
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) tc5::mbar_init(bar0 + 8 * i, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  // the stage's rows, s on, of the first array; the second's follow array_bytes on
  __device__ __forceinline__ const uint8_t* rows_of(int stage, int64_t s) const {
    return data + (uint32_t)(stage * ARRAYS) * array_bytes +
           (WIDE ? 0u : (uint32_t)(s * row_bytes) & 15u);
  }
  __device__ __forceinline__ void issue(int stage, int64_t s) const {
    const int64_t from = (s * row_bytes) & ~int64_t(15);
    int64_t to = ((s + R) * row_bytes + 15) & ~int64_t(15);
    if (to > total) to = total & ~int64_t(15);
    const uint32_t bar = bar0 + 8 * stage, bytes = to > from ? (uint32_t)(to - from) : 0u;
    tc5::mbar_arrive_tx(bar, bytes * ARRAYS);
    if (bytes)
#pragma unroll
      for (int i = 0; i < ARRAYS; ++i)
        tc5::bulk_load(tc5::smem_u32(data) + (stage * ARRAYS + i) * array_bytes, src[i] + from,
                       bytes, bar);
  }
  __device__ __forceinline__ void wait(int stage, uint32_t parity) {
    if (!dead) dead = !tc5::mbar_wait(bar0 + 8 * stage, parity, &g_norm_error);
  }
  // The array's last bytes into the stage of its last rows, s on.
  __device__ __forceinline__ void patch(int stage, int64_t s) const {
    if (WIDE || (s + R) * row_bytes < total || (total & 15) == 0) return;
    const int64_t from = (s * row_bytes) & ~int64_t(15), cut = max(total & ~int64_t(15), from);
    if ((int)threadIdx.x < (int)(total - cut))
      for (int i = 0; i < ARRAYS; ++i)
        data[(stage * ARRAYS + i) * array_bytes + (cut - from) + threadIdx.x] =
            src[i][cut + threadIdx.x];
    __syncthreads();
  }
};

// The E columns of a row that a thread owns, in pairs: E / VW vectors of VW
// values, vector i at slot i G + t. VW is 16 bytes' worth where rows are
// multiples of 16 bytes, else two values or one (still 64 bytes or more a warp).
template <class T, int E_, int VW>
struct Own {
  using A = acc_t<T>;
  static constexpr int E = E_;
  static_assert(E % 2 == 0 && E % VW == 0, "whole pairs and vectors");
  int t, G, n_d;
  uint32_t off, step;      // bytes: the first column, and from one vector to the next
  __device__ __forceinline__ Own(int t_, int G_, int n_d_)
      : t(t_), G(G_), n_d(n_d_), off(t_ * VW * (int)sizeof(T)), step(G_ * VW * (int)sizeof(T)) {}
  __device__ __forceinline__ bool has(int e) const { return (e / VW * G + t) * VW < n_d; }
  __device__ __forceinline__ int col(int e) const { return (e / VW * G + t) * VW + e % VW; }
  // zeros where the thread has no column (a single vector: only called where
  // it has it)
  __device__ __forceinline__ void load(const uint8_t* row, Pair<A> (&o)[E / 2]) const {
    if constexpr (VW > 1) {
#pragma unroll
      for (int i = 0; i < E / VW; ++i) {
        Vec<T, VW> v;
        if (E > VW) {
#pragma unroll
          for (int k = 0; k < VW; ++k) v.v[k] = round_to<T>(A(0));
        }
        if (E == VW || has(i * VW)) v = *reinterpret_cast<const Vec<T, VW>*>(row + off + i * step);
#pragma unroll
        for (int k = 0; k < VW / 2; ++k)
          o[i * (VW / 2) + k] = widen2(*reinterpret_cast<const Vec<T, 2>*>(&v.v[2 * k]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const T* p = reinterpret_cast<const T*>(row + off + e * step);
        const T* q = reinterpret_cast<const T*>(row + off + (e + 1) * step);
        o[e / 2] = Pair<A>(has(e) ? load_acc<T>(*p) : A(0), has(e + 1) ? load_acc<T>(*q) : A(0));
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* row, const Pair<A> (&o)[E / 2]) const {
    if constexpr (VW > 1) {
#pragma unroll
      for (int i = 0; i < E / VW; ++i) {
        Vec<T, VW> v;
#pragma unroll
        for (int k = 0; k < VW / 2; ++k)
          *reinterpret_cast<Vec<T, 2>*>(&v.v[2 * k]) = narrow2<T>(o[i * (VW / 2) + k]);
        if (has(i * VW)) *reinterpret_cast<Vec<T, VW>*>(row + off + i * step) = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (has(e)) *reinterpret_cast<T*>(row + off + e * step) = round_to<T>(o[e / 2].lo());
        if (has(e + 1))
          *reinterpret_cast<T*>(row + off + (e + 1) * step) = round_to<T>(o[e / 2].hi());
      }
    }
  }
  // the pair with zeros where the thread has no column
  __device__ __forceinline__ Pair<A> only(int k, Pair<A> c) const {
    if (E == VW) return c;
    if (VW > 1) return has(2 * k) ? c : both(A(0));
    return Pair<A>(has(2 * k) ? c.lo() : A(0), has(2 * k + 1) ? c.hi() : A(0));
  }
  __device__ __forceinline__ void params(const A* p, A other, Pair<A> (&o)[E / 2]) const {
#pragma unroll
    for (int e = 0; e < E; e += 2)
      o[e / 2] = Pair<A>(p && has(e) ? p[col(e)] : other, p && has(e + 1) ? p[col(e + 1)] : other);
  }
  __device__ __forceinline__ void store_params(A* p, const Pair<A> (&o)[E / 2]) const {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      if (has(e)) p[col(e)] = o[e / 2].lo();
      if (has(e + 1)) p[col(e + 1)] = o[e / 2].hi();
    }
  }
};

template <class A>
__device__ __forceinline__ void clear_red(A (*red)[8][32]) {
  for (int i = threadIdx.x; i < 2 * 8 * 32; i += blockDim.x) (&red[0][0][0])[i] = A(0);
  __syncthreads();
}

// R rows a turn: what a turn costs beside its arithmetic (the wait, two
// barriers, the shuffles) is shared by them.
template <class T, int E, int VW, int R, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB)
ln_fwd_ring_kernel(const T* __restrict__ x, const acc_t<T>* __restrict__ w,
                   const acc_t<T>* __restrict__ b, T* __restrict__ y,
                   acc_t<T>* __restrict__ m_stack, acc_t<T>* __restrict__ r_stack, double eps,
                   int64_t n_s, int n_d, int stages) {
  using A = acc_t<T>;
  using O = Own<T, E, VW>;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ A red[2][8][32];
  Ring<T, 1, VW * sizeof(T) == 16> ring(sm, stages, R, n_d, n_s, x, nullptr);
  clear_red(red);
  const int t = threadIdx.x;
  const O own(t, (int)blockDim.x, n_d);
  Pair<A> wr[E / 2], br[E / 2];
  own.params(w, A(1), wr);
  own.params(b, A(0), br);
  const int64_t first = (int64_t)blockIdx.x * R, step = (int64_t)gridDim.x * R;
  if (t == 0)
    for (int i = 0; i < stages && first + i * step < n_s; ++i) ring.issue(i, first + i * step);
  int stage = 0;
  uint32_t parity = 0;
  const A inv = A(1) / (A)n_d;
  uint8_t* out = reinterpret_cast<uint8_t*>(y) + first * ring.row_bytes;
  const bool mine = own.has(0);
  for (int64_t s = first; s < n_s; s += step, out += step * ring.row_bytes) {
    const int rows = (int)min((int64_t)R, n_s - s);
    ring.wait(stage, parity);
    ring.patch(stage, s);
    const uint8_t* in = ring.rows_of(stage, s);
    Pair<A> c[R][E / 2];
    A v[R];
    // rows past the last one: whatever the stage holds, never stored
#pragma unroll
    for (int q = 0; q < R; ++q) {
      v[q] = 0;
      if (mine) {
        own.load(in + q * ring.row_bytes, c[q]);
        Pair<A> sum = c[q][0];
#pragma unroll
        for (int k = 1; k < E / 2; ++k) sum = add2(sum, c[q][k]);
        v[q] = sum.lo() + sum.hi();
      }
    }
    block_sums<R>(v, red, 0, [&](A z) { return z * inv; });
    // every thread has read the stage: it takes the rows to come
    if (t == 0 && s + stages * step < n_s) ring.issue(stage, s + stages * step);
    A mean[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = v[q];
      const Pair<A> minus = both(-v[q]);
      Pair<A> sq = both(A(0));
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        c[q][k] = add2(c[q][k], minus);
        const Pair<A> z = own.only(k, c[q][k]);
        sq = fma2(z, z, sq);
      }
      v[q] = mine ? sq.lo() + sq.hi() : A(0);
    }
    block_sums<R>(v, red, 1, [&](A z) { return A(1) / sqrt(z * inv + (A)eps); });
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) {
        const Pair<A> rstd = both(v[q]);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) c[q][k] = fma2(mul2(c[q][k], rstd), wr[k], br[k]);
        own.store(out + q * ring.row_bytes, c[q]);
      }
    if (t < rows) {
      A a = mean[0], z = v[0];
#pragma unroll
      for (int q = 1; q < R; ++q)
        if (t == q) a = mean[q], z = v[q];
      m_stack[s + t] = a;
      r_stack[s + t] = z;
    }
    if (++stage == stages) stage = 0, parity ^= 1;
  }
}

// KEEP: h and g w stay in registers over the sums; otherwise the row is read
// and widened from the stage once more (the longest rows, whose threads have 80
// registers and spill 100 to 324 bytes: 4096 x 12288 bf16 110 us, 46 by memory).
// 16-bit rows wait for a turn's two sums and their barriers: with 16 warps an SM
// 47 % of the issue slots are used and 0.76 of the measured copy rate (16384 x
// 4096 bf16: 81 us, 61 by memory; 103 when the row is read twice). Float32 rows
// have twice the bytes to wait for: 125 us, 0.98 of that rate.
template <class T, int E, int VW, int R, int MAXT, bool KEEP>
__global__ void __launch_bounds__(MAXT, 1)
ln_bwd_ring_kernel(BwdArgs p, int stages) {
  using A = acc_t<T>;
  using O = Own<T, E, VW>;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ A red[2][8][32];
  Ring<T, 2, VW * sizeof(T) == 16> ring(sm, stages, R, p.n_d, p.n_s, p.x, p.yb);
  clear_red(red);
  const int t = threadIdx.x;
  const O own(t, (int)blockDim.x, p.n_d);
  const A* m = (const A*)p.m;
  const A* r = (const A*)p.r;
  Pair<A> w[E / 2], sw[E / 2], sb[E / 2];
  own.params((const A*)p.w, A(1), w);
#pragma unroll
  for (int k = 0; k < E / 2; ++k) sw[k] = sb[k] = both(A(0));
  const int64_t first = (int64_t)blockIdx.x * R, step = (int64_t)gridDim.x * R;
  if (t == 0)
    for (int i = 0; i < stages && first + i * step < p.n_s; ++i) ring.issue(i, first + i * step);
  int stage = 0, turn = 0, last = -1;
  uint32_t parity = 0;
  const A inv = A(1) / (A)p.n_d;
  A nr[R], nm[R];                 // the next turn's statistics, loaded a turn ahead
  auto stats = [&](int64_t s) {
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (s + q < p.n_s) nr[q] = r[s + q], nm[q] = m[s + q];
  };
  stats(first);
  int64_t out = first * ring.row_bytes;
  // a thread past the row's end has nothing to do (single columns: some of them)
  const bool mine = own.has(0);
  for (int64_t s = first; s < p.n_s; s += step, out += step * ring.row_bytes) {
    const int rows = (int)min((int64_t)R, p.n_s - s);
    // h = (x - mean) rstd: one product with -mean rstd added is an instruction
    // less, but its rounding does not cancel where the mean is large for the row
    A rstd[R], less[R], v[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      rstd[q] = nr[q];
      less[q] = -nm[q];
      v[2 * q] = v[2 * q + 1] = A(0);
    }
    stats(s + step);
    ring.wait(stage, parity);
    ring.patch(stage, s);
    const uint8_t* in = ring.rows_of(stage, s);
    Pair<A> kh[KEEP ? R : 1][E / 2], kg[KEEP ? R : 1][E / 2];
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) {
        Pair<A> cx[E / 2], cy[E / 2], sg = both(A(0)), sgh = both(A(0));
        own.load(in + q * ring.row_bytes, cx);
        own.load(in + ring.array_bytes + q * ring.row_bytes, cy);
        const Pair<A> rs = both(rstd[q]), mn = both(less[q]);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          // columns the thread does not have: yb = 0 there, so nothing is added
          const Pair<A> h = mul2(add2(cx[k], mn), rs), gw = mul2(cy[k], w[k]);
          sg = add2(sg, gw);
          sgh = fma2(gw, h, sgh);
          sw[k] = fma2(cy[k], h, sw[k]);
          sb[k] = add2(sb[k], cy[k]);
          if (KEEP) kh[KEEP ? q : 0][k] = h, kg[KEEP ? q : 0][k] = gw;
        }
        v[2 * q] = sg.lo() + sg.hi();
        v[2 * q + 1] = sgh.lo() + sgh.hi();
      }
    block_sums<2 * R>(v, red, turn, [&](A z) { return z * inv; });
    turn ^= 1;
    // every thread is past the previous turn's stage: it takes the rows to come
    if (t == 0 && last >= 0 && s + (stages - 1) * step < p.n_s)
      ring.issue(last, s + (stages - 1) * step);
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) {
        Pair<A> cx[E / 2], cy[E / 2];
        if (p.xb) {
          uint8_t* o = (uint8_t*)p.xb + out + q * ring.row_bytes;
          // rstd (g - mean(g) - h mean(g h))
          const Pair<A> rs = both(rstd[q]), mn = both(less[q]);
          const Pair<A> mg = both(-v[2 * q] * rstd[q]), mgh = both(-v[2 * q + 1] * rstd[q]);
          if (!KEEP) {
            own.load(in + q * ring.row_bytes, cx);
            own.load(in + ring.array_bytes + q * ring.row_bytes, cy);
          }
#pragma unroll
          for (int k = 0; k < E / 2; ++k) {
            const Pair<A> h = KEEP ? kh[KEEP ? q : 0][k] : mul2(add2(cx[k], mn), rs);
            const Pair<A> gw = KEEP ? kg[KEEP ? q : 0][k] : mul2(cy[k], w[k]);
            cx[k] = fma2(gw, rs, fma2(h, mgh, mg));
          }
          if (p.add) {
            own.load(o, cy);
#pragma unroll
            for (int k = 0; k < E / 2; ++k) cx[k] = add2(cx[k], cy[k]);
          }
          own.store(o, cx);
        }
        if (p.zero) {
#pragma unroll
          for (int k = 0; k < E / 2; ++k) cy[k] = both(A(0));
          own.store((uint8_t*)p.yb + out + q * ring.row_bytes, cy);
        }
      }
    last = stage;
    if (++stage == stages) stage = 0, parity ^= 1;
  }
  if (!p.sums) return;
  A* part = (A*)p.part + (int64_t)blockIdx.x * 2 * p.n_d;
  own.store_params(part, sw);
  own.store_params(part + p.n_d, sb);
}

// ---- a warp per row --------------------------------------------------------------------
constexpr int kRowWarps = 8;

// R rows a turn, all their loads in flight. Lanes with more than 16 bytes of a
// row take one row a turn and leave room for three blocks an SM (65536 x 512
// bf16: 34 us; 44 with two rows). Lanes with three vectors of 16-bit values (rows
// of 513 to 767) spill 120 to 136 bytes here and 200 to 236 in reverse, Float64
// rows of 129 to 191 200 to 220 there: 16384 x 640 bf16 19 and 36 us, 6.4 and 9.6
// by memory.
template <class T, int E, int VW, int R>
__global__ void __launch_bounds__(32 * kRowWarps, R == 1 ? 3 : 1)
ln_fwd_warp_kernel(const T* __restrict__ x, const acc_t<T>* __restrict__ w,
                   const acc_t<T>* __restrict__ b, T* __restrict__ y,
                   acc_t<T>* __restrict__ m_stack, acc_t<T>* __restrict__ r_stack, double eps,
                   int64_t n_s, int n_d) {
  using A = acc_t<T>;
  using O = Own<T, E, VW>;
  const int t = threadIdx.x & 31;
  const O own(t, 32, n_d);
  const int64_t row_bytes = n_d * (int64_t)sizeof(T);
  Pair<A> wr[E / 2], br[E / 2];
  own.params(w, A(1), wr);
  own.params(b, A(0), br);
  const bool mine = own.has(0);
  const A inv = A(1) / (A)n_d;
  const int64_t step = (int64_t)gridDim.x * kRowWarps * R;
  for (int64_t s = ((int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * R; s < n_s; s += step) {
    const uint8_t* in = reinterpret_cast<const uint8_t*>(x) + s * row_bytes;
    uint8_t* out = reinterpret_cast<uint8_t*>(y) + s * row_bytes;
    const int rows = (int)min((int64_t)R, n_s - s);
    Pair<A> c[R][E / 2];
    A v[R];
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) own.load(in + q * row_bytes, c[q]);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      v[q] = 0;
      if (q < rows && mine) {
        Pair<A> sum = c[q][0];
#pragma unroll
        for (int k = 1; k < E / 2; ++k) sum = add2(sum, c[q][k]);
        v[q] = sum.lo() + sum.hi();
      }
    }
    warp_sums<R>(v, [&](A z) { return z * inv; });
    A mean[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = v[q];
      v[q] = 0;
      if (q < rows && mine) {
        const Pair<A> minus = both(-mean[q]);
        Pair<A> sq = both(A(0));
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          c[q][k] = add2(c[q][k], minus);
          const Pair<A> z = own.only(k, c[q][k]);
          sq = fma2(z, z, sq);
        }
        v[q] = sq.lo() + sq.hi();
      }
    }
    warp_sums<R>(v, [&](A z) { return A(1) / sqrt(z * inv + (A)eps); });
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows) {
        if (mine) {
          const Pair<A> rstd = both(v[q]);
#pragma unroll
          for (int k = 0; k < E / 2; ++k) c[q][k] = fma2(mul2(c[q][k], rstd), wr[k], br[k]);
          own.store(out + q * row_bytes, c[q]);
        }
        if (t == 0) {
          m_stack[s + q] = mean[q];
          r_stack[s + q] = v[q];
        }
      }
  }
}

// blocks an SM that a lane's columns leave registers for
template <class T, int E> constexpr int bwd_warp_blocks() {
  return E <= 8 ? 4 : sizeof(T) == 4 ? 3 : 2;
}
template <class T, int E, int VW, int R>
__global__ void __launch_bounds__(32 * kRowWarps, (bwd_warp_blocks<T, E>()))
ln_bwd_warp_kernel(BwdArgs p) {
  using A = acc_t<T>;
  using O = Own<T, E, VW>;
  const int t = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const O own(t, 32, p.n_d);
  const int64_t row_bytes = p.n_d * (int64_t)sizeof(T);
  const A* m = (const A*)p.m;
  const A* r = (const A*)p.r;
  Pair<A> w[E / 2], sw[E / 2], sb[E / 2];
  own.params((const A*)p.w, A(1), w);
#pragma unroll
  for (int k = 0; k < E / 2; ++k) sw[k] = sb[k] = both(A(0));
  const bool mine = own.has(0);
  const A inv = A(1) / (A)p.n_d;
  const int64_t step = (int64_t)gridDim.x * kRowWarps * R;
  for (int64_t s = ((int64_t)blockIdx.x * kRowWarps + warp) * R; s < p.n_s; s += step) {
    const int rows = (int)min((int64_t)R, p.n_s - s);
    const int64_t at = s * row_bytes;
    Pair<A> cx[R][E / 2], cy[R][E / 2];     // x and yb, then h and g w
    A rstd[R], v[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) {
        own.load((const uint8_t*)p.x + at + q * row_bytes, cx[q]);
        own.load((const uint8_t*)p.yb + at + q * row_bytes, cy[q]);
      }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      rstd[q] = q < rows ? r[s + q] : A(0);
      const A less = q < rows ? -m[s + q] : A(0);
      v[2 * q] = v[2 * q + 1] = A(0);
      if (q < rows && mine) {
        Pair<A> sg = both(A(0)), sgh = both(A(0));
        const Pair<A> rs = both(rstd[q]), mn = both(less);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          // columns the lane does not have: yb = 0 there, so nothing is added
          const Pair<A> h = mul2(add2(cx[q][k], mn), rs), g = cy[q][k], gw = mul2(g, w[k]);
          sg = add2(sg, gw);
          sgh = fma2(gw, h, sgh);
          sw[k] = fma2(g, h, sw[k]);
          sb[k] = add2(sb[k], g);
          cx[q][k] = h;
          cy[q][k] = gw;
        }
        v[2 * q] = sg.lo() + sg.hi();
        v[2 * q + 1] = sgh.lo() + sgh.hi();
      }
    }
    warp_sums<2 * R>(v, [&](A z) { return z * inv; });
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows && mine) {
        if (p.xb) {
          uint8_t* o = (uint8_t*)p.xb + at + q * row_bytes;
          const Pair<A> rs = both(rstd[q]);
          const Pair<A> mg = both(-v[2 * q] * rstd[q]), mgh = both(-v[2 * q + 1] * rstd[q]);
#pragma unroll
          for (int k = 0; k < E / 2; ++k) cx[q][k] = fma2(cy[q][k], rs, fma2(cx[q][k], mgh, mg));
          if (p.add) {
            own.load(o, cy[q]);
#pragma unroll
            for (int k = 0; k < E / 2; ++k) cx[q][k] = add2(cx[q][k], cy[q][k]);
          }
          own.store(o, cx[q]);
        }
        if (p.zero) {
#pragma unroll
          for (int k = 0; k < E / 2; ++k) cy[q][k] = both(A(0));
          own.store((uint8_t*)p.yb + at + q * row_bytes, cy[q]);
        }
      }
  }
  if (!p.sums) return;
  // the block's warps, added in order
  extern __shared__ __align__(128) uint8_t sm[];
  A* part = reinterpret_cast<A*>(sm);       // 2 x n_d
  for (int q = 0; q < kRowWarps; ++q) {
    if (warp == q)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (own.has(e)) {
          const int d = own.col(e);
          const A a = e % 2 ? sw[e / 2].hi() : sw[e / 2].lo();
          const A z = e % 2 ? sb[e / 2].hi() : sb[e / 2].lo();
          part[d] = q ? part[d] + a : a;
          part[p.n_d + d] = q ? part[p.n_d + d] + z : z;
        }
    __syncthreads();
  }
  A* out = (A*)p.part + (int64_t)blockIdx.x * 2 * p.n_d;
  for (int d = threadIdx.x; d < 2 * p.n_d; d += 32 * kRowWarps) out[d] = part[d];
}

// wb and bb from the partials [count][2][n_d]: 32 columns a block, 32 warps
// that each add every 32nd partial, then the warps' sums in order.
template <class A>
__global__ void __launch_bounds__(1024)
ln_finish_kernel(const A* __restrict__ part, int count, int64_t n_d, A* __restrict__ wb,
                 A* __restrict__ bb, bool add) {
  __shared__ A sm[32][33];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + lane;    // 0 .. 2 n_d - 1: wb, then bb
  A acc = 0;
  if (d < 2 * n_d)
    acc = ordered_sum(part + d + (int64_t)warp * 2 * n_d, (count - warp + 31) / 32, 64 * n_d);
  sm[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || d >= 2 * n_d) return;
  A s = 0;
#pragma unroll
  for (int q = 0; q < 32; ++q) s += sm[q][lane];
  A* o = d < n_d ? (wb ? wb + d : nullptr) : (bb ? bb + d - n_d : nullptr);
  if (o) *o = add ? *o + s : s;
}

// ---- rows too long for registers ---------------------------------------------------
constexpr int kThreads = 256;

template <class T>
__global__ void __launch_bounds__(kThreads)
ln_fwd_long_kernel(const T* __restrict__ x, const acc_t<T>* __restrict__ w,
                   const acc_t<T>* __restrict__ b, T* __restrict__ y,
                   acc_t<T>* __restrict__ m_stack, acc_t<T>* __restrict__ r_stack, double eps,
                   int64_t n_d) {
  using A = acc_t<T>;
  __shared__ A red[kThreads / 32];
  const int64_t s = blockIdx.x;
  const T* xr = x + s * n_d;
  A sum = 0;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) sum += load_acc<T>(xr[d]);
  const A mean = block_sum(sum, red) / (A)n_d;
  A sq = 0;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) {
    const A c = load_acc<T>(xr[d]) - mean;
    sq += c * c;
  }
  const A rstd = A(1) / sqrt(block_sum(sq, red) / (A)n_d + (A)eps);
  if (threadIdx.x == 0) {
    m_stack[s] = mean;
    r_stack[s] = rstd;
  }
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) {
    const A h = (load_acc<T>(xr[d]) - mean) * rstd;
    y[s * n_d + d] = round_to<T>(h * (w ? w[d] : A(1)) + (b ? b[d] : A(0)));
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
ln_bwd_x_long_kernel(const T* __restrict__ x, T* __restrict__ xb, const acc_t<T>* __restrict__ w,
                     const T* __restrict__ yb, const acc_t<T>* __restrict__ m_stack,
                     const acc_t<T>* __restrict__ r_stack, int64_t n_d, bool add) {
  using A = acc_t<T>;
  __shared__ A red[kThreads / 32];
  const int64_t s = blockIdx.x, o = s * n_d;
  const A mean = m_stack[s], rstd = r_stack[s];
  A sg = 0, sgh = 0;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) {
    const A g = load_acc<T>(yb[o + d]) * (w ? w[d] : A(1));
    sg += g;
    sgh += g * ((load_acc<T>(x[o + d]) - mean) * rstd);
  }
  const A mg = block_sum(sg, red) / (A)n_d;
  const A mgh = block_sum(sgh, red) / (A)n_d;
  for (int64_t d = threadIdx.x; d < n_d; d += kThreads) {
    const A g = load_acc<T>(yb[o + d]) * (w ? w[d] : A(1));
    const A h = (load_acc<T>(x[o + d]) - mean) * rstd;
    const A v = rstd * (g - mg - h * mgh);
    xb[o + d] = round_to<T>(add ? load_acc<T>(xb[o + d]) + v : v);
  }
}

// Partial sums over a chunk of rows, one thread per column.
template <class T>
__global__ void __launch_bounds__(kThreads)
ln_bwd_w_long_kernel(const T* __restrict__ x, T* __restrict__ yb,
                     const acc_t<T>* __restrict__ m_stack, const acc_t<T>* __restrict__ r_stack,
                     int64_t n_s, int64_t n_d, int64_t rows, acc_t<T>* __restrict__ part,
                     bool zero) {
  using A = acc_t<T>;
  const int64_t d = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (d >= n_d) return;
  const int64_t s0 = blockIdx.y * rows, s1 = min(n_s, s0 + rows);
  A w = 0, b = 0;
  for (int64_t s = s0; s < s1; ++s) {
    const A v = load_acc<T>(yb[s * n_d + d]);
    w += v * ((load_acc<T>(x[s * n_d + d]) - m_stack[s]) * r_stack[s]);
    b += v;
    if (zero) yb[s * n_d + d] = round_to<T>(A(0));
  }
  part[(2 * (int64_t)blockIdx.y) * n_d + d] = w;
  part[(2 * (int64_t)blockIdx.y + 1) * n_d + d] = b;
}

// ---- which kernel --------------------------------------------------------------------
// Blocks of the reverse sweep, and so partials of the sums over rows.
constexpr int64_t kBwdBlocks = 148 * 8;

// Calls f(VW): what the rows' alignment allows an access to be.
template <class T, class F>
stade_status with_width(int align, F&& f) {
  using std::integral_constant;
  if (align >= 16) return f(integral_constant<int, 16 / (int)sizeof(T)>{});
  if constexpr (sizeof(T) < 8)
    if (align >= 2 * (int)sizeof(T)) return f(integral_constant<int, 2>{});
  return f(integral_constant<int, 1>{});
}

// Rows of less than 96 times 16 bytes go to a warp each: calls f(E, VW), E the
// columns of a lane. Vectors of 16 bytes only where most lanes get one.
template <class T, class F>
stade_status with_row_warps(int64_t n_d, int align, F&& f) {
  using std::integral_constant;
  constexpr int V = 16 / (int)sizeof(T);
  if (align >= 16 && n_d < 24 * V) align = n_d < 48 ? (int)sizeof(T) : 2 * (int)sizeof(T);
  return with_width<T>(align, [&](auto vw) {
    constexpr int VW = decltype(vw)::value;
    const int64_t per = (n_d + 32 * VW - 1) / (32 * VW) * VW;       // columns of a lane
    if constexpr (VW <= 2 && V >= 4)
      if (per <= 2) return f(integral_constant<int, 2>{}, vw);
    if constexpr (VW <= 4 && V == 8)
      if (per <= 4) return f(integral_constant<int, 4>{}, vw);
    if (per <= V) return f(integral_constant<int, V>{}, vw);
    if (per <= 2 * V) return f(integral_constant<int, 2 * V>{}, vw);
    return f(integral_constant<int, 3 * V>{}, vw);
  });
}

// Ring kernels: a block of `threads` threads a row (m vectors each), `rows` rows
// a turn, `stages` turns in flight, as many blocks an SM as registers and 200
// KB of shared memory allow.
//  - Forward: rows of up to 256 vectors one a thread and up to four rows a turn,
//    1,024 threads an SM at 64 registers; longer ones two vectors a thread and
//    two rows a turn, 640 threads at 96 (16384 x 4096 bf16: 49.6 us against 55.8
//    with one vector; 16384 x 2048: 34.9 against 31.0). Where that leaves blocks
//    of 257 to 384 threads with whole vectors, two of them and a row a turn do
//    better (8192 x 5000 f16: 43.8 against 46.3 us; single columns, 8192 x 4999:
//    76 against 64).
//  - Reverse: the row's h and g w stay in registers, 512 threads at 128, so two
//    vectors a thread and two or more blocks an SM rather than several rows a
//    turn, which left one block and its barriers alone on the SM (16384 x 4096
//    bf16: 83 us against 106 with four rows a turn; 32768 x 1024: 48 against
//    56). Narrower columns spill at two vectors' worth: one vector's and two rows
//    a turn there (32768 x 1023 bf16: 63 us against 93); 16-bit rows of 513 to
//    768 vectors' length one vector's and one row (8192 x 4999 f16: 94 against
//    133).
constexpr int kRingSmem = 205 * 1024;   // a block's ring, at most
struct RingPlan {
  int m, rows, threads, stages, blocks;
  size_t smem;
};
bool ring_plan(int64_t n_s, int64_t row_bytes, int size, bool rev, bool wide, RingPlan* p) {
  const int64_t slots = (row_bytes + 15) / 16;   // a thread owns 16 bytes of a row, or 32
  if (slots < 96 || slots > 2 * 768) return false;
  const int64_t single = rev ? (wide ? 0 : size == 2 ? 768 : 512) : 256;
  p->m = slots <= single ? 1 : 2;
  p->threads = (int)(((slots + p->m - 1) / p->m + 31) / 32 * 32);
  const bool two_blocks = !rev && wide && p->threads > 256 && p->threads <= 384;
  const int per_sm =
      two_blocks ? 2 : std::max(1, (rev ? 512 : p->m == 2 ? 640 : 1024) / p->threads);
  const int arrays = rev ? 2 : 1;
  const int64_t room = 200 * 1024 / (per_sm * row_bytes * arrays);   // rows in flight a block
  // several rows a turn where every block still gets two turns
  const bool one = n_s < 4 * 148 * per_sm || room < 4 || two_blocks || p->threads > 512 ||
                   (p->m > 1 && rev);
  p->rows = one ? 1 : p->m == 1 && !rev && room >= 8 && n_s >= 8 * 148 * per_sm ? 4 : 2;
  p->stages = (int)std::min<int64_t>(kMaxStages, std::max<int64_t>(2, room / p->rows));
  p->smem = 128 + p->stages * arrays * ((p->rows * row_bytes + 31) & ~int64_t(15));
  p->blocks = (int)std::min<int64_t>((n_s + p->rows - 1) / p->rows, 148 * per_sm);
  return p->smem <= kRingSmem;
}
// The limit of a kernel's shared memory is the kernel's, not the launch's: always
// the same value, so that host threads with rows of other lengths do not lower
// it between this call's setting and its launch.
template <class K>
stade_status allow_ring(K kern) {
  STADE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
  return STADE_OK;
}

template <class T>
stade_status fwd(const void* x, const void* w, const void* b, void* y, void* m, void* r, double eps,
                 int64_t n_s, int64_t n_d, cudaStream_t st) {
  using A = acc_t<T>;
  constexpr int V = 16 / (int)sizeof(T);
  const int align = row_align(n_d * sizeof(T), {x, y});
  const int64_t row_bytes = n_d * (int64_t)sizeof(T), slots = (row_bytes + 15) / 16;
  if (slots < 96)
    return with_row_warps<T>(n_d, align, [&](auto ee, auto vw) {
      constexpr int E = decltype(ee)::value, R = E <= V ? 4 : 1;
      const int64_t turns = (n_s + R * kRowWarps - 1) / (R * kRowWarps);
      ln_fwd_warp_kernel<T, E, decltype(vw)::value, R>
          <<<(unsigned)std::min<int64_t>(turns, 148 * (R == 1 ? 3 : 8)),
             32 * kRowWarps, 0, st>>>(
              (const T*)x, (const A*)w, (const A*)b, (T*)y, (A*)m, (A*)r, eps, n_s, (int)n_d);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  RingPlan rp;
  if (row_align(16, {x}) == 16 && ring_plan(n_s, row_bytes, sizeof(T), false, align == 16, &rp)) {
    return with_width<T>(align, [&](auto vw) {
      constexpr int VW = decltype(vw)::value;
      auto kern = rp.threads > 512 ? ln_fwd_ring_kernel<T, 2 * V, VW, 1, 768, 1>
                  : rp.m == 2 ? (rp.rows == 2 ? ln_fwd_ring_kernel<T, 2 * V, VW, 2, 512, 1>
                                 : rp.threads <= 384 ? ln_fwd_ring_kernel<T, 2 * V, VW, 1, 384, 2>
                                                     : ln_fwd_ring_kernel<T, 2 * V, VW, 1, 512, 1>)
                  : rp.rows == 4 ? ln_fwd_ring_kernel<T, V, VW, 4, 256, 4>
                  : rp.rows == 2 ? ln_fwd_ring_kernel<T, V, VW, 2, 256, 4>
                                 : ln_fwd_ring_kernel<T, V, VW, 1, 256, 4>;
      const stade_status ok = allow_ring(kern);
      if (ok != STADE_OK) return ok;
      kern<<<rp.blocks, rp.threads, rp.smem, st>>>((const T*)x, (const A*)w, (const A*)b, (T*)y,
                                                   (A*)m, (A*)r, eps, n_s, (int)n_d, rp.stages);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  }
  void (*kern)(const T*, const A*, const A*, T*, A*, A*, double, int) = nullptr;
  int threads = 0;
  if (n_d <= 1024) kern = ln_fwd_kernel<T, 128, 8>, threads = 128;
  else if (n_d <= 4096) kern = ln_fwd_kernel<T, 512, 8>, threads = 512;
  else if (n_d <= 8192) kern = ln_fwd_kernel<T, 1024, 8>, threads = 1024;
  if (kern)
    kern<<<(unsigned)n_s, threads, 0, st>>>((const T*)x, (const A*)w, (const A*)b, (T*)y, (A*)m,
                                            (A*)r, eps, (int)n_d);
  else
    ln_fwd_long_kernel<T><<<(unsigned)n_s, kThreads, 0, st>>>(
        (const T*)x, (const A*)w, (const A*)b, (T*)y, (A*)m, (A*)r, eps, n_d);
  STADE_CHECK_LAUNCH();
  return STADE_OK;
}

template <class T>
stade_status bwd(const void* x, void* xb, const void* w, void* wb, void* bb, void* yb,
                 const void* m, const void* r, int64_t n_s, int64_t n_d, void* ws, bool add,
                 bool zero, cudaStream_t st) {
  using A = acc_t<T>;
  const bool sums = wb || bb;
  if (!xb && !sums && !zero) return STADE_OK;
  constexpr int V = 16 / (int)sizeof(T);
  const int align = row_align(n_d * sizeof(T), {x, xb, yb});
  const int64_t row_bytes = n_d * (int64_t)sizeof(T), slots = (row_bytes + 15) / 16;
  int count = 0;
  RingPlan rp;
  stade_status e = STADE_OK;
  if (slots < 96) {
    e = with_row_warps<T>(n_d, align, [&](auto ee, auto vw) {
      constexpr int E = decltype(ee)::value, R = E <= V / 2 ? 2 : 1;
      const int64_t turns = (n_s + R * kRowWarps - 1) / (R * kRowWarps);
      count = (int)std::min<int64_t>(turns, 148 * bwd_warp_blocks<T, E>());
      const BwdArgs p{x, w, m, r, xb, yb, ws, n_s, (int)n_d, add, zero, sums};
      ln_bwd_warp_kernel<T, E, decltype(vw)::value, R>
          <<<count, 32 * kRowWarps, 2 * n_d * sizeof(A), st>>>(p);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  } else if (row_align(16, {x, yb}) == 16 && ring_plan(n_s, row_bytes, sizeof(T), true, align == 16, &rp)) {
    count = rp.blocks;
    const BwdArgs p{x, w, m, r, xb, yb, ws, n_s, (int)n_d, add, zero, sums};
    e = with_width<T>(align, [&](auto vw) {
      constexpr int VW = decltype(vw)::value;
      void (*kern)(BwdArgs, int) = ln_bwd_ring_kernel<T, 2 * V, VW, 1, 512, true>;
      if (rp.threads > 512) kern = ln_bwd_ring_kernel<T, 2 * V, VW, 1, 768, false>;
      if constexpr (VW != V)
        if (rp.m == 1)
          kern = rp.threads > 512 ? ln_bwd_ring_kernel<T, V, VW, 1, 768, true>
                 : rp.rows == 2   ? ln_bwd_ring_kernel<T, V, VW, 2, 512, true>
                                  : ln_bwd_ring_kernel<T, V, VW, 1, 512, true>;
      const stade_status ok = allow_ring(kern);
      if (ok != STADE_OK) return ok;
      kern<<<rp.blocks, rp.threads, rp.smem, st>>>(p, rp.stages);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  } else if (n_d <= 4096) {
    const BwdArgs p{x, w, m, r, xb, yb, ws, n_s, (int)n_d, add, zero, sums};
    const int threads = n_d <= 512 ? 128 : n_d <= 1024 ? 256 : n_d <= 2048 ? 512 : 1024;
    auto kern = threads == 128 ? ln_bwd_kernel<T, 128, 4>
                : threads == 256 ? ln_bwd_kernel<T, 256, 4>
                : threads == 512 ? ln_bwd_kernel<T, 512, 4> : ln_bwd_kernel<T, 1024, 4>;
    count = (int)std::min<int64_t>(n_s, 148 * (1024 / threads));
    kern<<<count, threads, 0, st>>>(p);
    STADE_CHECK_LAUNCH();
  } else {
    if (xb) {
      ln_bwd_x_long_kernel<T><<<(unsigned)n_s, kThreads, 0, st>>>(
          (const T*)x, (T*)xb, (const A*)w, (const T*)yb, (const A*)m, (const A*)r, n_d, add);
      STADE_CHECK_LAUNCH();
    }
    count = (int)std::min<int64_t>(n_s, 148);
    const int64_t rows = (n_s + count - 1) / count;
    const dim3 grid(ceil_div_u(n_d, kThreads), count);
    ln_bwd_w_long_kernel<T><<<grid, kThreads, 0, st>>>((const T*)x, (T*)yb, (const A*)m,
                                                       (const A*)r, n_s, n_d, rows, (A*)ws, zero);
    STADE_CHECK_LAUNCH();
  }
  if (e != STADE_OK || !sums) return e;
  return launch_next(ln_finish_kernel<A>, ceil_div_u(2 * n_d, 32), 1024, 0, st, (const A*)ws, count,
                     n_d, (A*)wb, (A*)bb, add);
}

stade_status check_sizes(const char* who, int dtype, int64_t n_s, int64_t n_d) {
  STADE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  STADE_REQUIRE(n_s >= 0 && n_d >= 0, "%s: negative size", who);
  STADE_REQUIRE(n_s < (int64_t(1) << 31) && n_d < (int64_t(1) << 31), "%s: size overflow", who);
  return STADE_OK;
}

}  // namespace

int norm_take_error() {
  int host = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&host, g_norm_error, sizeof(int)) != cudaSuccess) return -1;
  if (host) cudaMemcpyToSymbol(g_norm_error, &zero, sizeof(int));
  return host;
}

}  // namespace stade

using namespace stade;

extern "C" stade_status stade_layer_norm(int dtype, const void* x, const void* w, const void* b,
                                         void* y, void* m_stack, void* r_stack, double eps,
                                         int64_t n_s, int64_t n_d, const stade_opts* opts) {
  stade_status st = check_sizes("layer_norm", dtype, n_s, n_d);
  if (st != STADE_OK) return st;
  STADE_REQUIRE(eps >= 0, "layer_norm: eps must not be negative");
  if (n_s == 0 || n_d == 0) return STADE_OK;
  STADE_REQUIRE(x && y && m_stack && r_stack, "layer_norm: null array argument");
  cudaStream_t s = stream_of(opts);
  PhaseScope ph("layer_norm", s);
  return with_dtype(dtype, [&](auto t) {
    return fwd<decltype(t)>(x, w, b, y, m_stack, r_stack, eps, n_s, n_d, s);
  });
}

extern "C" size_t stade_layer_norm_b_workspace(int dtype, int64_t n_s, int64_t n_d) {
  if (n_s <= 0 || n_d <= 0) return 0;
  Sizer z;
  z.take<char>((size_t)std::min(n_s, kBwdBlocks) * 2 * n_d * (dtype == STADE_F64 ? 8 : 4));
  return z.bytes();
}

extern "C" stade_status stade_layer_norm_b(int dtype, const void* x, void* xb, const void* w,
                                           void* wb, void* bb, void* yb, const void* m_stack,
                                           const void* r_stack, int64_t n_s, int64_t n_d,
                                           const stade_opts* opts) {
  stade_status st = check_sizes("layer_norm_b", dtype, n_s, n_d);
  if (st != STADE_OK) return st;
  cudaStream_t s = stream_of(opts);
  const bool add = accumulates(opts);
  if (n_s == 0 || n_d == 0) {
    // no rows: the sums are empty
    if (!add && n_d > 0 && wb)
      STADE_CUDA(cudaMemsetAsync(wb, 0, n_d * (dtype == STADE_F64 ? 8 : 4), s));
    if (!add && n_d > 0 && bb)
      STADE_CUDA(cudaMemsetAsync(bb, 0, n_d * (dtype == STADE_F64 ? 8 : 4), s));
    return STADE_OK;
  }
  STADE_REQUIRE(x && yb && m_stack && r_stack, "layer_norm_b: null array argument");
  void* ws = nullptr;
  st = get_workspace(opts, stade_layer_norm_b_workspace(dtype, n_s, n_d), &ws);
  if (st != STADE_OK) return st;
  PhaseScope ph("layer_norm_b", s);
  return with_dtype(dtype, [&](auto t) {
    return bwd<decltype(t)>(x, xb, w, wb, bb, yb, m_stack, r_stack, n_s, n_d, ws, add,
                            consumes(opts), s);
  });
}
