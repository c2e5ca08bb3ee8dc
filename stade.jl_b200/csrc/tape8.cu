// The 8-bit tape: activation checkpoints as int8 codes with one power-of-two
// scale per 32 values of a row, the activations whose forward writes it and
// whose reverse sweep reads it.
//
//   top = max |x| of the group, k = floor(log2 top), e = max(k - 6, -126)
//   q = clip(rint(x 2^-e), -127, 127),   x^ = q 2^e
//   forward  y = f(x);    reverse  xb += yb f'(x^)
//
// The scale is a power of two, so x 2^-e and q 2^e are exact: the codes
// depend on x alone, not on the order or the precision of any arithmetic,
// and x^ is exact in every one of the types (7 bits of magnitude). Values
// below the top 1/128 of the group's binade are within 2^e / 2 of x, those
// above it within 2^e. The scale byte holds e + 127 (1 .. 248); 255 marks a group with an
// infinity or a NaN, which reads back as NaN throughout, so that an overflow
// in the forward shows in the gradient instead of vanishing in a code.
//
// Bound by memory, with the instructions close behind: gelu of 8192 x 8192 in
// bf16 takes 68 us forward and 67 us in reverse, 51 us each by their bytes, with
// three quarters of the issue slots in use; tanh in reverse 53 us. In Float32,
// 8192 x 4096: relu, tanh and silu 0.86 to 0.98 of the measured copy rate, gelu
// 55 us forward and 82 in reverse, 46 by their bytes (erff and expf).

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "token_ops.cuh"

namespace stade {
namespace {

constexpr int kGroup = 32;
constexpr int kThreads = 256;

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// Scale byte of a group from its largest magnitude; 255 for inf and NaN.
__device__ __forceinline__ int scale_code(float top) {
  const int bits = __float_as_int(top);          // top >= 0
  if (bits >= 0x7f800000) return 255;
  const int k = (bits >> 23) - 127;              // a subnormal gives -127: clipped below
  const int e = k - 6 < -126 ? -126 : k - 6;
  return e + 127;
}
__device__ __forceinline__ float restore(int q, int code) {
  return code == 255 ? __int_as_float(0x7fffffff) : (float)q * pow2f(code - 127);
}

// ---- activations -------------------------------------------------------------------
// f(x) and f'(x) with CUDA's erff, expf and tanhf, for Float32 arrays.
template <int ACT>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == STADE_ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
  if constexpr (ACT == STADE_ACT_TANH) return tanhf(x);
  if constexpr (ACT == STADE_ACT_SILU) return x / (1.f + expf(-x));
  if constexpr (ACT == STADE_ACT_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  return x;
}
// relu: max(x, 0)' = (1 + sign x) / 2, the partial of the generated sweeps
template <int ACT>
__device__ __forceinline__ float act_df(float x) {
  if constexpr (ACT == STADE_ACT_RELU) return x > 0.f ? 1.f : x < 0.f ? 0.f : x == 0.f ? 0.5f : x;
  if constexpr (ACT == STADE_ACT_TANH) {
    const float h = tanhf(x);
    return 1.f - h * h;
  }
  if constexpr (ACT == STADE_ACT_SILU) {
    const float p = 1.f / (1.f + expf(-x));
    return p * (1.f + x * (1.f - p));
  }
  if constexpr (ACT == STADE_ACT_GELU)
    return 0.5f * (1.f + erff(x * 0.70710678118654752f)) +
           x * expf(-0.5f * x * x) * 0.39894228040143268f;
  return 1.f;
}

// The same for 16-bit arrays, at two special-function instructions an element and
// two elements an instruction elsewhere. With erff and expf a gelu step of 8192
// x 8192 in bf16 was bound by its instructions (213 us; memory alone 103 us).
// Values and slopes keep their relative precision in the tails, where they fall
// off as exp(-|x|) or exp(-x^2 / 2): 2e-6, and 1e-5 where the exponential's
// argument is near -126 and its rounding counts; half a unit in the last place
// of the types is 2e-3 and 2.4e-4. (The Float32 forms above follow the formulas
// as they stand, 1 + erf and 1 - tanh^2: within 1e-7 of 1 + |x|.)
using P2 = Pair<float>;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.44269504088896340736f;

// q = 1 - Phi(|x|) and g = exp(-x^2 / 2). q / g is a smooth function of |x| that
// falls from 1/2 as 1 / |x|: a polynomial in t = 1 / (1 + 0.362 |x|) without a
// constant term, fitted to the smallest relative error over 0 .. 13.5 (beyond
// that g is 0 in Float32): 1.1e-6 in Float32 arithmetic. A term less is 4.1e-6,
// twice half a unit of f16 where the slope passes through 0, for 1.4 us of the
// reverse sweep of 8192 x 8192.
__device__ __forceinline__ P2 tail2(P2 x, P2* g) {
  constexpr float c = 0.362f;
  const P2 t(rcp(fmaf(fabsf(x.lo()), c, 1.f)), rcp(fmaf(fabsf(x.hi()), c, 1.f)));
  const P2 s = mul2(mul2(x, x), both(-0.5f * kLog2e));
  *g = P2(ex2(s.lo()), ex2(s.hi()));
  P2 p = fma2(both(0.0480388179f), t, both(-0.180348381f));
  p = fma2(p, t, both(0.177071109f));
  p = fma2(p, t, both(0.0285237320f));
  p = fma2(p, t, both(0.139540404f));
  p = fma2(p, t, both(0.142669395f));
  p = fma2(p, t, both(0.144505307f));
  return mul2(mul2(p, t), *g);
}
// 1 / (1 + exp(-x)), which reaches 0 where exp(-x) passes Float32's range: x
// times any floor would not vanish for the largest x
__device__ __forceinline__ P2 sigmoid2(P2 x) {
  return P2(rcp(1.f + ex2(x.lo() * -kLog2e)), rcp(1.f + ex2(x.hi() * -kLog2e)));
}
// 1 - 2 / (1 + exp 2x), and the Taylor polynomial near 0, where that cancels
__device__ __forceinline__ P2 tanh2(P2 x) {
  const P2 s = mul2(x, x);
  P2 p = fma2(s, both(-17.f / 315.f), both(2.f / 15.f));
  p = fma2(s, p, both(-1.f / 3.f));
  const P2 small = mul2(x, fma2(s, p, both(1.f)));
  const float a = fmaf(rcp(1.f + ex2(fminf(x.lo() * (2.f * kLog2e), 120.f))), -2.f, 1.f);
  const float b = fmaf(rcp(1.f + ex2(fminf(x.hi() * (2.f * kLog2e), 120.f))), -2.f, 1.f);
  // a NaN takes the polynomial, which passes it on
  return P2(s.lo() >= 0.0625f ? a : small.lo(), s.hi() >= 0.0625f ? b : small.hi());
}

template <int ACT>
__device__ __forceinline__ P2 act_f2(P2 x) {
  if constexpr (ACT == STADE_ACT_TANH) return tanh2(x);
  if constexpr (ACT == STADE_ACT_SILU) {
    return mul2(x, sigmoid2(x));
  }
  if constexpr (ACT == STADE_ACT_GELU) {
    // x Phi(x) = max(x, 0) - |x| (1 - Phi(|x|)). The product is 0 from 14 on; to
    // the right also for an infinity, to the left it is NaN there, as x times
    // (1 + erf) is in the Float32 form.
    P2 g;
    const P2 q = tail2(x, &g);
    return P2(fmaf(-fabsf(fminf(x.lo(), 14.f)), q.lo(), fmaxf(x.lo(), 0.f)),
              fmaf(-fabsf(fminf(x.hi(), 14.f)), q.hi(), fmaxf(x.hi(), 0.f)));
  }
  return P2(act_f<ACT>(x.lo()), act_f<ACT>(x.hi()));
}
template <int ACT>
__device__ __forceinline__ P2 act_df2(P2 x) {
  if constexpr (ACT == STADE_ACT_TANH) {
    // 1 - tanh^2 = 4 r (1 - r), r = 1 / (1 + exp 2|x|): no cancellation
    const P2 r(rcp(1.f + ex2(fabsf(x.lo()) * (2.f * kLog2e))),
               rcp(1.f + ex2(fabsf(x.hi()) * (2.f * kLog2e))));
    return mul2(mul2(r, both(4.f)), fma2(r, both(-1.f), both(1.f)));
  }
  if constexpr (ACT == STADE_ACT_SILU) {
    const P2 p = sigmoid2(x);
    return mul2(p, fma2(x, fma2(p, both(-1.f), both(1.f)), both(1.f)));
  }
  if constexpr (ACT == STADE_ACT_GELU) {
    P2 g;
    const P2 q = tail2(x, &g);
    const P2 o = fma2(q, both(-1.f), both(1.f));
    const P2 c(x.lo() < 0.f ? q.lo() : o.lo(), x.hi() < 0.f ? q.hi() : o.hi());   // Phi(x)
    return fma2(mul2(x, both(0.39894228040143268f)), g, c);
  }
  return P2(act_df<ACT>(x.lo()), act_df<ACT>(x.hi()));
}
template <int ACT, bool FAST> __device__ __forceinline__ P2 act_pair(P2 x) {
  if constexpr (FAST) return act_f2<ACT>(x);
  return P2(act_f<ACT>(x.lo()), act_f<ACT>(x.hi()));
}
template <int ACT, bool FAST> __device__ __forceinline__ P2 act_d_pair(P2 x) {
  if constexpr (FAST) return act_df2<ACT>(x);
  return P2(act_df<ACT>(x.lo()), act_df<ACT>(x.hi()));
}

// Adding 1.5 2^23 rounds a value of less than 2^22 to the nearest whole number,
// ties to even, and leaves it in the low bits: the code's byte is the low one.
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ P2 code_bits2(P2 v, P2 inv) {
  const P2 r = mul2(v, inv);
  return add2(P2(fminf(fmaxf(r.lo(), -127.f), 127.f), fminf(fmaxf(r.hi(), -127.f), 127.f)),
              both(kMagic));
}
__device__ __forceinline__ uint32_t pack4(P2 a, P2 b) {
  return __byte_perm(__byte_perm(__float_as_uint(a.lo()), __float_as_uint(a.hi()), 0x0040),
                     __byte_perm(__float_as_uint(b.lo()), __float_as_uint(b.hi()), 0x0040), 0x5410);
}
// Bytes k and k + 1 of w, biased by 128 (w = codes ^ 0x80808080), times step:
// 2^23 + byte has the byte in its low bits; all of it exact (the difference
// first: 2^23 step passes Float32's range where step is its largest).
__device__ __forceinline__ P2 code_value2(uint32_t w, int k, P2 step) {
  const P2 f(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + k)),
             __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + k + 1)));
  return mul2(add2(f, both(-8388736.f)), step);
}

// A thread takes V = 8 values of a row, four threads a group: 16 to 32 bytes
// of x a load, 8 bytes of codes a store, and the group's largest magnitude by
// two shuffles. Rows that are no multiple of 8 values, or arrays that do not
// start on the boundary such accesses need, go through the kernels further
// down.
constexpr int kV = 8;

template <class T>
struct alignas(16) Eight {
  T v[kV];
};
// 8 values as the array holds them: one access of 16 bytes, or two of them.
template <class T> __device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> r;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<int4*>(&r) = *reinterpret_cast<const int4*>(p);
  } else {
    reinterpret_cast<int4*>(&r)[0] = reinterpret_cast<const int4*>(p)[0];
    reinterpret_cast<int4*>(&r)[1] = reinterpret_cast<const int4*>(p)[1];
  }
  return r;
}
template <class T> __device__ __forceinline__ P2 pair_of(const Eight<T>& r, int k) {
  return widen2(reinterpret_cast<const Vec<T, 2>*>(&r)[k]);
}
template <class T> __device__ __forceinline__ void store8(T* p, const P2 (&v)[4]) {
  Eight<T> r;
#pragma unroll
  for (int k = 0; k < 4; ++k) reinterpret_cast<Vec<T, 2>*>(&r)[k] = narrow2<T>(v[k]);
  reinterpret_cast<int4*>(p)[0] = reinterpret_cast<const int4*>(&r)[0];
  if constexpr (sizeof(T) == 4)
    reinterpret_cast<int4*>(p)[1] = reinterpret_cast<const int4*>(&r)[1];
}
// Largest magnitude of 8 values, NaN if one is.
__device__ __forceinline__ float top8(const Eight<float>& r) {
  uint32_t m = 0;        // magnitudes are ordered as whole numbers, NaN above infinity
#pragma unroll
  for (int k = 0; k < kV; ++k)
    m = max(m, reinterpret_cast<const uint32_t*>(&r)[k] & 0x7fffffffu);
  return __uint_as_float(m);
}
template <class T2>
__device__ __forceinline__ T2 top2(const T2* r) {
  return __hmax2_nan(__hmax2_nan(__habs2(r[0]), __habs2(r[1])),
                     __hmax2_nan(__habs2(r[2]), __habs2(r[3])));
}
__device__ __forceinline__ float top8(const Eight<__nv_bfloat16>& r) {
  const __nv_bfloat162 m = top2(reinterpret_cast<const __nv_bfloat162*>(&r));
  return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
__device__ __forceinline__ float top8(const Eight<__half>& r) {
  const __half2 m = top2(reinterpret_cast<const __half2*>(&r));
  return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
// The larger of two magnitudes, a NaN above all.
__device__ __forceinline__ float larger(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

// Rows of n8 eights, thread i of `count`, 4 n_g a row: a row's last group may
// have threads past its end.
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
push8_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ q,
             uint8_t* __restrict__ e, uint32_t n8, uint32_t n_g, int64_t count) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const bool live = i < count;
  // the usual case, rows of whole groups, needs no division
  int64_t at = i;
  bool in = live;
  if (n8 != 4 * n_g) {
    const int64_t s = i / (4 * n_g);
    const uint32_t c = (uint32_t)(i - s * (4 * n_g));
    in = live && c < n8;
    at = s * n8 + c;
  }
  Eight<T> v;
  float top = 0.f;
  if (in) {
    v = load8<T>(x + at * kV);
    top = top8(v);
  }
  top = larger(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = larger(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int code = scale_code(top);
  if (in) {
    const float inv = pow2f(127 - min(code, 253));
    P2 p[4], c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p[k] = pair_of<T>(v, k);
      c[k] = code_bits2(p[k], both(inv));
    }
    uint2 w = make_uint2(pack4(c[0], c[1]), pack4(c[2], c[3]));
    if (code == 255) w = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(q + at * kV) = w;
    if constexpr (ACT != STADE_ACT_NONE) {
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = act_pair<ACT, sizeof(T) == 2>(p[k]);
      store8<T>(y + at * kV, p);
    }
  }
  if (live && (threadIdx.x & 3) == 0) e[i >> 2] = (uint8_t)code;
}

// 16-bit arrays: held to 32 registers, eight blocks an SM (gelu takes 34 without
// that, and 78 us instead of 68 for 8192 x 8192).
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 1)
pop8_kernel(T* __restrict__ xb, T* __restrict__ yb, const int8_t* __restrict__ q,
            const uint8_t* __restrict__ e, uint32_t n8, uint32_t n_g, int64_t count, bool add,
            bool zero) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  int64_t group = i >> 2;
  if (n8 != 4 * n_g) {
    const int64_t s = i / n8;
    group = s * n_g + (uint32_t)(i - s * n8) / 4;
  }
  uint2 w = *reinterpret_cast<const uint2*>(q + i * kV);
  Eight<T> g;
  if constexpr (ACT != STADE_ACT_NONE) g = load8<T>(yb + i * kV);
  const int code = e[group];
  w.x ^= 0x80808080u;
  w.y ^= 0x80808080u;
  const float step = code == 255 ? __int_as_float(0x7fffffff) : pow2f(code - 127);
  const P2 step2 = both(step);
  P2 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = code_value2(k < 2 ? w.x : w.y, 2 * (k % 2), step2);
  if constexpr (ACT == STADE_ACT_NONE) {
    store8<T>(xb + i * kV, v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = mul2(pair_of<T>(g, k), act_d_pair<ACT, sizeof(T) == 2>(v[k]));
    if (add) {
      const Eight<T> old = load8<T>(xb + i * kV);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = add2(v[k], pair_of<T>(old, k));
    }
    store8<T>(xb + i * kV, v);
    if (zero) {
      P2 z[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
      store8<T>(yb + i * kV, z);
    }
  }
}

// Other row lengths and alignments: a warp takes kGroups groups of a row, all of
// them in flight. W = 2 (rows of an even number of values): half a warp a
// group, two neighbours a lane; W = 1: a warp a group, a value a lane, two
// groups at a time, so that arithmetic runs in pairs either way.
constexpr int kGroups = 8;
constexpr int kPairs = kGroups / 2;

// Where a lane's pair k lies in a row, from the first of the groups on: its two
// values, and the two groups they belong to.
template <int W>
struct Place {
  int lane;
  __device__ __forceinline__ int group(int k, int v) const {
    return W == 2 ? 2 * k + (lane >> 4) : 2 * k + v;
  }
  __device__ __forceinline__ int value(int k, int v) const {
    return group(k, v) * kGroup + (W == 2 ? 2 * (lane & 15) + v : lane);
  }
};
template <int W, class E>
__device__ __forceinline__ Vec<E, 2> load_pair(const E* p, const Place<W>& pl, int k,
                                               int64_t left) {
  Vec<E, 2> r{};
  if constexpr (W == 2) {
    if (pl.value(k, 0) < left) r = *reinterpret_cast<const Vec<E, 2>*>(p + pl.value(k, 0));
  } else {
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (pl.value(k, v) < left) r.v[v] = p[pl.value(k, v)];
  }
  return r;
}
template <int W, class E>
__device__ __forceinline__ void store_pair(E* p, const Place<W>& pl, int k, int64_t left,
                                           Vec<E, 2> r) {
  if constexpr (W == 2) {
    if (pl.value(k, 0) < left) *reinterpret_cast<Vec<E, 2>*>(p + pl.value(k, 0)) = r;
  } else {
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (pl.value(k, v) < left) p[pl.value(k, v)] = r.v[v];
  }
}

template <class T, int ACT, int W>
__global__ void __launch_bounds__(kThreads)
push_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ q,
            uint8_t* __restrict__ e, int64_t n_g, int64_t segs, int64_t count, int64_t n_d) {
  const int lane = threadIdx.x & 31;
  const Place<W> pl{lane};
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < count;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = i / segs, g0 = (i - s * segs) * kGroups;
    const int64_t at = s * n_d + g0 * kGroup, left = n_d - g0 * kGroup;
    Vec<T, 2> raw[kPairs];
#pragma unroll
    for (int k = 0; k < kPairs; ++k) raw[k] = load_pair<W>(x + at, pl, k, left);
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const P2 v = widen2(raw[k]);
      int code[2];
      if constexpr (W == 2) {
        float top = larger(v.lo(), v.hi());
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o));
        code[0] = code[1] = scale_code(top);
      } else {
        code[0] = scale_code(__uint_as_float(
            __reduce_max_sync(0xffffffffu, __float_as_uint(v.lo()) & 0x7fffffffu)));
        code[1] = scale_code(__uint_as_float(
            __reduce_max_sync(0xffffffffu, __float_as_uint(v.hi()) & 0x7fffffffu)));
      }
      const P2 inv(pow2f(127 - min(code[0], 253)), pow2f(127 - min(code[1], 253)));
      const P2 c = code_bits2(v, inv);
      Vec<int8_t, 2> w;
      w.v[0] = code[0] == 255 ? 0 : (int8_t)(__float_as_uint(c.lo()) & 255u);
      w.v[1] = code[1] == 255 ? 0 : (int8_t)(__float_as_uint(c.hi()) & 255u);
      store_pair<W>(q + at, pl, k, left, w);
      if constexpr (ACT != STADE_ACT_NONE)
        store_pair<W>(y + at, pl, k, left, narrow2<T>(act_pair<ACT, sizeof(T) == 2>(v)));
      // one lane a group: the half warp's first, or lanes 0 and 1
      const int v1 = W == 2 ? 0 : lane & 1;
      const int g = pl.group(k, v1);
      if ((W == 2 ? (lane & 15) == 0 : lane < 2) && g0 + g < n_g)
        e[s * n_g + g0 + g] = (uint8_t)(v1 ? code[1] : code[0]);
    }
  }
}

// ACT none: x = x^ (pop). Otherwise xb (+)= yb f'(x^).
template <class T, int ACT, int W>
__global__ void __launch_bounds__(kThreads)
pop_kernel(T* __restrict__ xb, T* __restrict__ yb, const int8_t* __restrict__ q,
           const uint8_t* __restrict__ e, int64_t n_g, int64_t segs, int64_t count, int64_t n_d,
           bool add, bool zero) {
  const int lane = threadIdx.x & 31;
  const Place<W> pl{lane};
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < count;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = i / segs, g0 = (i - s * segs) * kGroups;
    const int64_t at = s * n_d + g0 * kGroup, left = n_d - g0 * kGroup;
    const int codes = lane < kGroups && g0 + lane < n_g ? e[s * n_g + g0 + lane] : 0;
    Vec<int8_t, 2> c[kPairs];
    Vec<T, 2> g[kPairs], old[kPairs];
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      c[k] = load_pair<W>(q + at, pl, k, left);
      if constexpr (ACT != STADE_ACT_NONE) {
        g[k] = load_pair<W>((const T*)yb + at, pl, k, left);
        if (add) old[k] = load_pair<W>((const T*)xb + at, pl, k, left);
      }
    }
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const int code0 = __shfl_sync(0xffffffffu, codes, pl.group(k, 0));
      const int code1 = W == 2 ? code0 : __shfl_sync(0xffffffffu, codes, pl.group(k, 1));
      const P2 v(restore(c[k].v[0], code0), restore(c[k].v[1], code1));
      if constexpr (ACT == STADE_ACT_NONE) {
        store_pair<W>(xb + at, pl, k, left, narrow2<T>(v));
      } else {
        P2 r = mul2(widen2(g[k]), act_d_pair<ACT, sizeof(T) == 2>(v));
        if (add) r = add2(r, widen2(old[k]));
        store_pair<W>(xb + at, pl, k, left, narrow2<T>(r));
        if (zero) store_pair<W>(yb + at, pl, k, left, narrow2<T>(both(0.f)));
      }
    }
  }
}

template <class F>
stade_status with_type(int dtype, F&& f) {
  if (dtype == STADE_F32) return f(float{});
  if (dtype == STADE_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}
template <class F>
stade_status with_act(int act, F&& f) {
  using std::integral_constant;
  switch (act) {
    case STADE_ACT_RELU: return f(integral_constant<int, STADE_ACT_RELU>{});
    case STADE_ACT_TANH: return f(integral_constant<int, STADE_ACT_TANH>{});
    case STADE_ACT_SILU: return f(integral_constant<int, STADE_ACT_SILU>{});
    case STADE_ACT_GELU: return f(integral_constant<int, STADE_ACT_GELU>{});
    default: return f(integral_constant<int, STADE_ACT_NONE>{});
  }
}

unsigned blocks_for(int64_t warps) {
  const int64_t b = (warps + kThreads / 32 - 1) / (kThreads / 32);
  return (unsigned)std::min<int64_t>(b, 148 * 8 * 16);
}

unsigned blocks8(int64_t count) {
  return (unsigned)((count + kThreads - 1) / kThreads);
}

stade_status check_args(const char* who, int dtype, int act, int64_t n_s, int64_t n_d) {
  STADE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  if (dtype == STADE_F64)
    return fail(STADE_ENOTSUP, "%s: the 8-bit tape holds Float32 and 16-bit values", who);
  STADE_REQUIRE(act >= STADE_ACT_NONE && act <= STADE_ACT_GELU, "%s: bad activation %d", who, act);
  int64_t n;
  STADE_REQUIRE(n_s >= 0 && n_d >= 0, "%s: negative size", who);
  STADE_REQUIRE(mul_ok(n_s, n_d, &n), "%s: size overflow", who);
  return STADE_OK;
}

stade_status push(const char* who, int dtype, int act, const void* x, void* y, int8_t* q,
                  uint8_t* e, int64_t n_s, int64_t n_d, const stade_opts* opts) {
  stade_status st = check_args(who, dtype, act, n_s, n_d);
  if (st != STADE_OK) return st;
  if (n_s == 0 || n_d == 0) return STADE_OK;
  STADE_REQUIRE(x && q && e && (y || act == STADE_ACT_NONE), "%s: null array argument", who);
  cudaStream_t s = stream_of(opts);
  PhaseScope ph(who, s);
  const int64_t n_g = (n_d + kGroup - 1) / kGroup;
  // 8 values of every array in whole accesses
  const bool eights = n_d % kV == 0 && row_align(16, {x, y}) == 16 && row_align(8, {q}) >= 8 &&
                      n_d < (int64_t(1) << 31) && n_s * n_g < (int64_t(1) << 36);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      if (eights) {
        const int64_t count = n_s * n_g * 4;
        push8_kernel<T, decltype(a)::value><<<blocks8(count), kThreads, 0, s>>>(
            (const T*)x, (T*)y, q, e, (uint32_t)(n_d / kV), (uint32_t)n_g, count);
        STADE_CHECK_LAUNCH();
        return (stade_status)STADE_OK;
      }
      const int64_t segs = (n_g + kGroups - 1) / kGroups;
      const bool even = n_d % 2 == 0 && row_align(2 * sizeof(T), {x, y}) >= 2 * (int)sizeof(T) &&
                        row_align(2, {q}) >= 2;
      constexpr int ACT = decltype(a)::value;
      auto kern = even ? push_kernel<T, ACT, 2> : push_kernel<T, ACT, 1>;
      kern<<<blocks_for(n_s * segs), kThreads, 0, s>>>((const T*)x, (T*)y, q, e, n_g, segs,
                                                       n_s * segs, n_d);
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  });
}

stade_status pop(const char* who, int dtype, int act, void* xb, void* yb, const int8_t* q,
                 const uint8_t* e, int64_t n_s, int64_t n_d, const stade_opts* opts) {
  stade_status st = check_args(who, dtype, act, n_s, n_d);
  if (st != STADE_OK) return st;
  if (n_s == 0 || n_d == 0) return STADE_OK;
  STADE_REQUIRE(xb && q && e && (yb || act == STADE_ACT_NONE), "%s: null array argument", who);
  cudaStream_t s = stream_of(opts);
  PhaseScope ph(who, s);
  const int64_t n_g = (n_d + kGroup - 1) / kGroup;
  const bool eights = n_d % kV == 0 && row_align(16, {xb, yb}) == 16 && row_align(8, {q}) >= 8 &&
                      n_d < (int64_t(1) << 31) && n_s * n_g < (int64_t(1) << 36);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      if (eights) {
        const int64_t count = n_s * n_d / kV;
        pop8_kernel<T, decltype(a)::value><<<blocks8(count), kThreads, 0, s>>>(
            (T*)xb, (T*)yb, q, e, (uint32_t)(n_d / kV), (uint32_t)n_g, count, accumulates(opts),
            consumes(opts));
        STADE_CHECK_LAUNCH();
        return (stade_status)STADE_OK;
      }
      const int64_t segs = (n_g + kGroups - 1) / kGroups;
      const bool even = n_d % 2 == 0 && row_align(2 * sizeof(T), {xb, yb}) >= 2 * (int)sizeof(T) &&
                        row_align(2, {q}) >= 2;
      constexpr int ACT = decltype(a)::value;
      auto kern = even ? pop_kernel<T, ACT, 2> : pop_kernel<T, ACT, 1>;
      kern<<<blocks_for(n_s * segs), kThreads, 0, s>>>((T*)xb, (T*)yb, q, e, n_g, segs, n_s * segs,
                                                       n_d, accumulates(opts), consumes(opts));
      STADE_CHECK_LAUNCH();
      return (stade_status)STADE_OK;
    });
  });
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" int64_t stade_initstacks_tape8(int64_t n_s, int64_t n_d) {
  return n_s <= 0 || n_d <= 0 ? 0 : n_s * ((n_d + kGroup - 1) / kGroup);
}

extern "C" stade_status stade_tape8_push(int dtype, const void* x, int8_t* q_stack,
                                         uint8_t* e_stack, int64_t n_s, int64_t n_d,
                                         const stade_opts* opts) {
  return push("tape8_push", dtype, STADE_ACT_NONE, x, nullptr, q_stack, e_stack, n_s, n_d, opts);
}

extern "C" stade_status stade_tape8_pop(int dtype, void* x, const int8_t* q_stack,
                                        const uint8_t* e_stack, int64_t n_s, int64_t n_d,
                                        const stade_opts* opts) {
  return pop("tape8_pop", dtype, STADE_ACT_NONE, x, nullptr, q_stack, e_stack, n_s, n_d, opts);
}

extern "C" stade_status stade_act_tape8(int dtype, int act, const void* x, void* y, int8_t* q_stack,
                                        uint8_t* e_stack, int64_t n_s, int64_t n_d,
                                        const stade_opts* opts) {
  STADE_REQUIRE(act != STADE_ACT_NONE, "act_tape8: bad activation %d", act);
  return push("act_tape8", dtype, act, x, y, q_stack, e_stack, n_s, n_d, opts);
}

extern "C" stade_status stade_act_tape8_b(int dtype, int act, void* xb, void* yb,
                                          const int8_t* q_stack, const uint8_t* e_stack,
                                          int64_t n_s, int64_t n_d, const stade_opts* opts) {
  STADE_REQUIRE(act != STADE_ACT_NONE, "act_tape8_b: bad activation %d", act);
  return pop("act_tape8_b", dtype, act, xb, yb, q_stack, e_stack, n_s, n_d, opts);
}
