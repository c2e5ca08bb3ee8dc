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

#include <initializer_list>

#include "token_ops.cuh"

namespace stade {
namespace {

constexpr int kThreads = 256;

template <class T>
__global__ void __launch_bounds__(kThreads)
ln_fwd_kernel(const T* __restrict__ x, const acc_t<T>* __restrict__ w,
              const acc_t<T>* __restrict__ b, T* __restrict__ y, acc_t<T>* __restrict__ m_stack,
              acc_t<T>* __restrict__ r_stack, double eps, int64_t n_d) {
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
ln_bwd_x_kernel(const T* __restrict__ x, T* __restrict__ xb, const acc_t<T>* __restrict__ w,
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
ln_bwd_w_kernel(const T* __restrict__ x, T* __restrict__ yb, const acc_t<T>* __restrict__ m_stack,
                const acc_t<T>* __restrict__ r_stack, int64_t n_s, int64_t n_d, int64_t rows,
                acc_t<T>* __restrict__ part, bool zero) {
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
  part[(2 * blockIdx.y) * n_d + d] = w;
  part[(2 * blockIdx.y + 1) * n_d + d] = b;
}

template <class A>
__global__ void __launch_bounds__(kThreads)
ln_bwd_finish_kernel(const A* __restrict__ part, int count, int64_t n_d, A* __restrict__ wb,
                     A* __restrict__ bb, bool add) {
  const int64_t d = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (d >= n_d) return;
  if (wb) {
    const A s = ordered_sum(part + d, count, 2 * n_d);
    wb[d] = add ? wb[d] + s : s;
  }
  if (bb) {
    const A s = ordered_sum(part + n_d + d, count, 2 * n_d);
    bb[d] = add ? bb[d] + s : s;
  }
}

int row_chunks(int64_t n_s) { return (int)(n_s < 148 ? n_s : 148); }

template <class T>
stade_status fwd(const void* x, const void* w, const void* b, void* y, void* m, void* r, double eps,
                 int64_t n_s, int64_t n_d, cudaStream_t st) {
  using A = acc_t<T>;
  ln_fwd_kernel<T><<<(unsigned)n_s, kThreads, 0, st>>>(
      (const T*)x, (const A*)w, (const A*)b, (T*)y, (A*)m, (A*)r, eps, n_d);
  STADE_CHECK_LAUNCH();
  return STADE_OK;
}

template <class T>
stade_status bwd(const void* x, void* xb, const void* w, void* wb, void* bb, void* yb,
                 const void* m, const void* r, int64_t n_s, int64_t n_d, void* ws, bool add,
                 bool zero, cudaStream_t st) {
  using A = acc_t<T>;
  if (xb) {
    ln_bwd_x_kernel<T><<<(unsigned)n_s, kThreads, 0, st>>>(
        (const T*)x, (T*)xb, (const A*)w, (const T*)yb, (const A*)m, (const A*)r, n_d, add);
    STADE_CHECK_LAUNCH();
  }
  const int chunks = row_chunks(n_s);
  const int64_t rows = (n_s + chunks - 1) / chunks;
  const dim3 grid(ceil_div_u(n_d, kThreads), chunks);
  ln_bwd_w_kernel<T><<<grid, kThreads, 0, st>>>((const T*)x, (T*)yb, (const A*)m, (const A*)r, n_s,
                                                n_d, rows, (A*)ws, zero);
  STADE_CHECK_LAUNCH();
  ln_bwd_finish_kernel<A><<<ceil_div_u(n_d, kThreads), kThreads, 0, st>>>((const A*)ws, chunks, n_d,
                                                                         (A*)wb, (A*)bb, add);
  STADE_CHECK_LAUNCH();
  return STADE_OK;
}

stade_status check_sizes(const char* who, int dtype, int64_t n_s, int64_t n_d) {
  STADE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  STADE_REQUIRE(n_s >= 0 && n_d >= 0, "%s: negative size", who);
  STADE_REQUIRE(n_s < (int64_t(1) << 31) && n_d < (int64_t(1) << 31), "%s: size overflow", who);
  return STADE_OK;
}

}  // namespace
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
  z.take<char>((size_t)row_chunks(n_s) * 2 * n_d * (dtype == STADE_F64 ? 8 : 4));
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
