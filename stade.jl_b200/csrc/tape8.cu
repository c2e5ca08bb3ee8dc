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
// FAST (16-bit arrays): errors of a few 1e-7 of 1 + |x|, below a hundredth of
// what rounding the result costs, at two special-function instructions an
// element. With CUDA's erff, expf and tanhf a gelu step of 8192 x 8192 in bf16
// was bound by their instructions (213 us, 103 us by memory). Float32 arrays
// use those.

// 1 - Phi(z), z >= 0, and exp(-z^2 / 2): the rational approximation 7.1.26 of
// Abramowitz and Stegun for erfc(z / sqrt 2), error at most 1.5e-7.
__device__ __forceinline__ float tail_fast(float z, float* g) {
  const float t = __fdividef(1.f, fmaf(z, 0.3275911f * 0.70710678f, 1.f));
  const float p = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t,
                            -0.284496736f), t, 0.254829592f) * t;
  *g = __expf(-0.5f * z * z);
  return 0.5f * p * *g;
}
__device__ __forceinline__ float cdf_fast(float x, float* g) {
  const float q = tail_fast(fabsf(x), g);
  return x < 0.f ? q : 1.f - q;
}
// 1 - 2 / (1 + exp 2x), and the Taylor polynomial near 0, where that cancels
__device__ __forceinline__ float tanh_fast(float x) {
  const float s = x * x;
  const float small =
      x * fmaf(s, fmaf(s, fmaf(s, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  const float big = 1.f - __fdividef(2.f, 1.f + __expf(2.f * fminf(x, 40.f)));
  return s < 0.0625f ? small : big;
}
__device__ __forceinline__ float sigmoid_fast(float x) {
  return __fdividef(1.f, 1.f + __expf(fminf(-x, 80.f)));
}

template <int ACT, bool FAST>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == STADE_ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
  if constexpr (ACT == STADE_ACT_TANH) return FAST ? tanh_fast(x) : tanhf(x);
  if constexpr (ACT == STADE_ACT_SILU) return FAST ? x * sigmoid_fast(x) : x / (1.f + expf(-x));
  if constexpr (ACT == STADE_ACT_GELU) {
    float g;
    return FAST ? x * cdf_fast(x, &g) : 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  }
  return x;
}
// relu: max(x, 0)' = (1 + sign x) / 2, the partial of the generated sweeps
template <int ACT, bool FAST>
__device__ __forceinline__ float act_df(float x) {
  if constexpr (ACT == STADE_ACT_RELU) return x > 0.f ? 1.f : x < 0.f ? 0.f : x == 0.f ? 0.5f : x;
  if constexpr (ACT == STADE_ACT_TANH) {
    const float h = FAST ? tanh_fast(x) : tanhf(x);
    return 1.f - h * h;
  }
  if constexpr (ACT == STADE_ACT_SILU) {
    const float p = FAST ? sigmoid_fast(x) : 1.f / (1.f + expf(-x));
    return p * (1.f + x * (1.f - p));
  }
  if constexpr (ACT == STADE_ACT_GELU) {
    if (FAST) {
      float g;
      const float c = cdf_fast(x, &g);
      return fmaf(x * 0.39894228040143268f, g, c);
    }
    return 0.5f * (1.f + erff(x * 0.70710678118654752f)) +
           x * expf(-0.5f * x * x) * 0.39894228040143268f;
  }
  return 1.f;
}

// Adding 1.5 2^23 rounds a value of less than 2^22 to the nearest whole number,
// ties to even, and leaves it in the low bits: the code's byte is the low one.
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
  return __float_as_uint(fminf(fmaxf(v * inv, -127.f), 127.f) + kMagic);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte k of w, biased by 128 (w = codes ^ 0x80808080), times step.
__device__ __forceinline__ float code_value(uint32_t w, int k, float step) {
  const float f = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + k));   // 2^23 + byte
  return (f - 8388736.f) * step;
}

// A thread takes V = 8 values of a row, four threads a group: 16 to 32 bytes
// of x a load, 8 bytes of codes a store, and the group's largest magnitude by
// two shuffles. Rows that are no multiple of 8 values, or arrays that do not
// start on the boundary such accesses need, go through the kernels further
// down, one value a thread.
constexpr int kV = 8;

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[kV]) {
  if constexpr (sizeof(T) == 2) {
    const Vec<T, 8> r = *reinterpret_cast<const Vec<T, 8>*>(p);
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = load_acc<T>(r.v[k]);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 r = reinterpret_cast<const float4*>(p)[h];
      v[4 * h] = r.x; v[4 * h + 1] = r.y; v[4 * h + 2] = r.z; v[4 * h + 3] = r.w;
    }
  }
}
// Largest magnitude of 8 values, NaN if one is.
__device__ __forceinline__ float top8(const float* p, const float (&v)[kV]) {
  uint32_t m = 0;        // magnitudes are ordered as whole numbers, NaN above infinity
#pragma unroll
  for (int k = 0; k < kV; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  return __uint_as_float(m);
}
template <class T2>
__device__ __forceinline__ T2 top2(const T2* r) {
  return __hmax2_nan(__hmax2_nan(__habs2(r[0]), __habs2(r[1])),
                     __hmax2_nan(__habs2(r[2]), __habs2(r[3])));
}
__device__ __forceinline__ float top8(const __nv_bfloat16* p, const float (&)[kV]) {
  const int4 r = *reinterpret_cast<const int4*>(p);
  const __nv_bfloat162 m = top2(reinterpret_cast<const __nv_bfloat162*>(&r));
  return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
__device__ __forceinline__ float top8(const __half* p, const float (&)[kV]) {
  const int4 r = *reinterpret_cast<const int4*>(p);
  const __half2 m = top2(reinterpret_cast<const __half2*>(&r));
  return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
// The larger of two magnitudes, a NaN above all.
__device__ __forceinline__ float larger(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[kV]) {
  if constexpr (sizeof(T) == 2) {
    Vec<T, 8> r;
#pragma unroll
    for (int k = 0; k < kV; ++k) r.v[k] = round_to<T>(v[k]);
    *reinterpret_cast<Vec<T, 8>*>(p) = r;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      reinterpret_cast<float4*>(p)[h] =
          make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
  }
}

// Rows of n8 eights; thread i of `count` (a multiple of 4 a row: a row's last
// group may have threads past its end).
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
push8_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ q,
             uint8_t* __restrict__ e, uint32_t n8, uint32_t n_g, int64_t count) {
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads; i0 < count; i0 += (int64_t)gridDim.x * kThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool live = i < count;
    // the usual case, rows of whole groups, needs no division
    int64_t at = i, group = i >> 2;
    bool in = live;
    if (n8 != 4 * n_g) {
      const int64_t s = i / (4 * n_g);
      const uint32_t c = (uint32_t)(i - s * (4 * n_g));
      in = live && c < n8;
      at = s * n8 + c;
    }
    float v[kV];
    float top = 0.f;
    if (in) {
      load8<T>(x + at * kV, v);
      top = top8(x + at * kV, v);
    }
    top = larger(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = larger(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int code = scale_code(top);
    if (in) {
      const float inv = pow2f(127 - min(code, 253));
      uint32_t c[kV];
#pragma unroll
      for (int k = 0; k < kV; ++k) c[k] = code_bits(v[k], inv);
      uint2 w = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
      if (code == 255) w = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(q + at * kV) = w;
      if constexpr (ACT != STADE_ACT_NONE) {
#pragma unroll
        for (int k = 0; k < kV; ++k) v[k] = act_f<ACT, sizeof(T) == 2>(v[k]);
        store8<T>(y + at * kV, v);
      }
    }
    if (live && (threadIdx.x & 3) == 0) e[group] = (uint8_t)code;
  }
}

template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
pop8_kernel(T* __restrict__ xb, T* __restrict__ yb, const int8_t* __restrict__ q,
            const uint8_t* __restrict__ e, uint32_t n8, uint32_t n_g, int64_t count, bool add,
            bool zero) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * kThreads) {
    int64_t group = i >> 2;
    if (n8 != 4 * n_g) {
      const int64_t s = i / n8;
      group = s * n_g + (uint32_t)(i - s * n8) / 4;
    }
    const int code = e[group];
    uint2 w = *reinterpret_cast<const uint2*>(q + i * kV);
    w.x ^= 0x80808080u;
    w.y ^= 0x80808080u;
    const float step = code == 255 ? __int_as_float(0x7fffffff) : pow2f(code - 127);
    float v[kV], g[kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = code_value(k < 4 ? w.x : w.y, k % 4, step);
    if constexpr (ACT == STADE_ACT_NONE) {
      store8<T>(xb + i * kV, v);
    } else {
      load8<T>(yb + i * kV, g);
#pragma unroll
      for (int k = 0; k < kV; ++k) g[k] *= act_df<ACT, sizeof(T) == 2>(v[k]);
      if (add) {
        load8<T>(xb + i * kV, v);
#pragma unroll
        for (int k = 0; k < kV; ++k) g[k] += v[k];
      }
      store8<T>(xb + i * kV, g);
      if (zero) {
#pragma unroll
        for (int k = 0; k < kV; ++k) g[k] = 0.f;
        store8<T>(yb + i * kV, g);
      }
    }
  }
}

// Any row length and alignment: a warp takes kGroups groups of a row, a value a
// lane of each, all of them in flight.
constexpr int kGroups = 8;

template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
push_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ q,
            uint8_t* __restrict__ e, int64_t n_g, int64_t segs, int64_t count, int64_t n_d) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < count;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = i / segs, g0 = (i - s * segs) * kGroups;
    const int64_t at = s * n_d + g0 * kGroup + lane;
    const int64_t left = n_d - g0 * kGroup - lane;     // values of the row from this lane's on
    float v[kGroups];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
      v[j] = j * kGroup < left ? (float)load_acc<T>(x[at + j * kGroup]) : 0.f;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7fffffffu);
      const int code = scale_code(__uint_as_float(top));
      if (lane == j) mine = code;
      const uint32_t c = code == 255 ? 0u : code_bits(v[j], pow2f(127 - min(code, 253)));
      if (j * kGroup < left) {
        q[at + j * kGroup] = (int8_t)(c & 255u);
        if constexpr (ACT != STADE_ACT_NONE)
          y[at + j * kGroup] = round_to<T>(act_f<ACT, sizeof(T) == 2>(v[j]));
      }
    }
    if (lane < kGroups && g0 + lane < n_g) e[s * n_g + g0 + lane] = (uint8_t)mine;
  }
}

// ACT none: x = x^ (pop). Otherwise xb (+)= yb f'(x^).
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
pop_kernel(T* __restrict__ xb, T* __restrict__ yb, const int8_t* __restrict__ q,
           const uint8_t* __restrict__ e, int64_t n_g, int64_t segs, int64_t count, int64_t n_d,
           bool add, bool zero) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < count;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = i / segs, g0 = (i - s * segs) * kGroups;
    const int64_t at = s * n_d + g0 * kGroup + lane;
    const int64_t left = n_d - g0 * kGroup - lane;
    const int codes = lane < kGroups && g0 + lane < n_g ? e[s * n_g + g0 + lane] : 0;
    int8_t c[kGroups];
    float g[kGroups], old[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
      if (j * kGroup < left) {
        c[j] = q[at + j * kGroup];
        if constexpr (ACT != STADE_ACT_NONE) {
          g[j] = (float)load_acc<T>(yb[at + j * kGroup]);
          if (add) old[j] = (float)load_acc<T>(xb[at + j * kGroup]);
        }
      }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int code = __shfl_sync(0xffffffffu, codes, j);
      if (j * kGroup < left) {
        const float v = restore(c[j], code);
        if constexpr (ACT == STADE_ACT_NONE) {
          xb[at + j * kGroup] = round_to<T>(v);
        } else {
          float r = g[j] * act_df<ACT, sizeof(T) == 2>(v);
          if (add) r += old[j];
          xb[at + j * kGroup] = round_to<T>(r);
          if (zero) yb[at + j * kGroup] = round_to<T>(0.f);
        }
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
  const int64_t b = (count + kThreads - 1) / kThreads;
  return (unsigned)std::min<int64_t>(b, 148 * 8 * 16);
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

stade_status push(const char* who, int dtype, int act, const void* x, void* y, int8_t* q, uint8_t* e,
                  int64_t n_s, int64_t n_d, const stade_opts* opts) {
  stade_status st = check_args(who, dtype, act, n_s, n_d);
  if (st != STADE_OK) return st;
  if (n_s == 0 || n_d == 0) return STADE_OK;
  STADE_REQUIRE(x && q && e && (y || act == STADE_ACT_NONE), "%s: null array argument", who);
  cudaStream_t s = stream_of(opts);
  PhaseScope ph(who, s);
  const int64_t n_g = (n_d + kGroup - 1) / kGroup;
  // 8 values of every array in whole accesses
  const bool eights = n_d % kV == 0 && row_align(16, {x, y}) == 16 && row_align(8, {q}) >= 8 &&
                      n_d < (int64_t(1) << 31);
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
      push_kernel<T, decltype(a)::value><<<blocks_for(n_s * segs), kThreads, 0, s>>>(
          (const T*)x, (T*)y, q, e, n_g, segs, n_s * segs, n_d);
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
                      n_d < (int64_t(1) << 31);
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
      pop_kernel<T, decltype(a)::value><<<blocks_for(n_s * segs), kThreads, 0, s>>>(
          (T*)xb, (T*)yb, q, e, n_g, segs, n_s * segs, n_d, accumulates(opts), consumes(opts));
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
