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

#include <initializer_list>

#include "token_ops.cuh"

namespace stade {
namespace {

constexpr int kGroup = 32;
constexpr int kThreads = 256;

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// Scale exponent of a group from its largest magnitude; bad for inf and NaN.
struct Scale {
  uint8_t code;
  float inv;   // 2^-e, split in two factors below 2^127: inv * inv2
};
__device__ __forceinline__ int scale_code(float top) {
  const int bits = __float_as_int(top);          // top >= 0
  if (bits >= 0x7f800000) return 255;
  const int k = (bits >> 23) - 127;              // a subnormal gives -127: clipped below
  const int e = k - 6 < -126 ? -126 : k - 6;
  return e + 127;
}
__device__ __forceinline__ int quantise(float v, int code) {
  if (code == 255) return 0;
  const float r = rintf(v * pow2f(127 - code));  // 2^-e, e in -126 .. 121: a normal number
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}
__device__ __forceinline__ float restore(int q, int code) {
  return code == 255 ? __int_as_float(0x7fffffff) : (float)q * pow2f(code - 127);
}

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

// One warp per group of 32 values.
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
push_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ q,
            uint8_t* __restrict__ e, int64_t n_g, int64_t groups, int64_t n_d) {
  const int lane = threadIdx.x & 31;
  for (int64_t g = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < groups;
       g += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = g / n_g, d = (g % n_g) * kGroup + lane;
    const bool in = d < n_d;
    const float v = in ? (float)load_acc<T>(x[s * n_d + d]) : 0.f;
    unsigned top = __float_as_uint(fabsf(v));    // ordered as integers, NaN above infinity
    top = __reduce_max_sync(0xffffffffu, top);
    const int code = scale_code(__uint_as_float(top));
    if (in) {
      q[s * n_d + d] = (int8_t)quantise(v, code);
      if constexpr (ACT != STADE_ACT_NONE) y[s * n_d + d] = round_to<T>(act_f<ACT>(v));
    }
    if (lane == 0) e[g] = (uint8_t)code;
  }
}

// ACT none: x = x^ (pop). Otherwise xb (+)= yb f'(x^).
template <class T, int ACT>
__global__ void __launch_bounds__(kThreads)
pop_kernel(T* __restrict__ xb, T* __restrict__ yb, const int8_t* __restrict__ q,
           const uint8_t* __restrict__ e, int64_t n_g, int64_t groups, int64_t n_d, bool add,
           bool zero) {
  const int lane = threadIdx.x & 31;
  for (int64_t g = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < groups;
       g += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = g / n_g, d = (g % n_g) * kGroup + lane;
    if (d >= n_d) continue;
    const int64_t i = s * n_d + d;
    const float v = restore(q[i], e[g]);
    if constexpr (ACT == STADE_ACT_NONE) {
      xb[i] = round_to<T>(v);
    } else {
      float r = (float)load_acc<T>(yb[i]) * act_df<ACT>(v);
      if (add) r += (float)load_acc<T>(xb[i]);
      xb[i] = round_to<T>(r);
      if (zero) yb[i] = round_to<T>(0.f);
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

unsigned blocks_for(int64_t groups) {
  const int64_t b = (groups + kThreads / 32 - 1) / (kThreads / 32);
  return (unsigned)(b < 148 * 8 ? b : 148 * 8);
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
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      push_kernel<T, decltype(a)::value><<<blocks_for(n_s * n_g), kThreads, 0, s>>>(
          (const T*)x, (T*)y, q, e, n_g, n_s * n_g, n_d);
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
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      pop_kernel<T, decltype(a)::value><<<blocks_for(n_s * n_g), kThreads, 0, s>>>(
          (T*)xb, (T*)yb, q, e, n_g, n_s * n_g, n_d, accumulates(opts), consumes(opts));
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
