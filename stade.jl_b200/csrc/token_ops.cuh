// What the token-model operators (embed, layer_norm, tape8, expert_mm) share:
// element types, vector access, the two adjoint flags and argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace stade {

// Sums, statistics and parameter adjoints are held in Float32 for the 16-bit
// types (one rounding, when the result is stored) and in the type itself
// otherwise.
template <class T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
template <class T> using acc_t = typename AccOf<T>::type;

template <class T> __device__ __forceinline__ acc_t<T> load_acc(T v) { return v; }
template <> __device__ __forceinline__ float load_acc(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float load_acc(__half v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T round_to(acc_t<T> v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half round_to<__half>(float v) {
  return __float2half_rn(v);
}

// V consecutive elements moved as one load or store (V * sizeof(T) = 2 .. 16
// bytes, the address a multiple of that).
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// Two values of the sums' type computed on together: one instruction for two
// Float32 multiply-adds (fma.rn.f32x2), where the issue rate and not memory
// would bound a kernel on 16-bit data.
template <class A> struct Pair {
  A a, b;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(A x, A y) : a(x), b(y) {}
  __device__ __forceinline__ A lo() const { return a; }
  __device__ __forceinline__ A hi() const { return b; }
};
template <> struct Pair<float> {
  unsigned long long r;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float x, float y) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  }
  __device__ __forceinline__ float lo() const {
    return __uint_as_float((uint32_t)r);
  }
  __device__ __forceinline__ float hi() const {
    return __uint_as_float((uint32_t)(r >> 32));
  }
};
template <class A> __device__ __forceinline__ Pair<A> both(A x) { return Pair<A>(x, x); }
template <class A> __device__ __forceinline__ Pair<A> add2(Pair<A> x, Pair<A> y) {
  return Pair<A>(x.a + y.a, x.b + y.b);
}
template <class A> __device__ __forceinline__ Pair<A> mul2(Pair<A> x, Pair<A> y) {
  return Pair<A>(x.a * y.a, x.b * y.b);
}
template <class A> __device__ __forceinline__ Pair<A> fma2(Pair<A> x, Pair<A> y, Pair<A> z) {
  return Pair<A>(fma(x.a, y.a, z.a), fma(x.b, y.b, z.b));
}
template <> __device__ __forceinline__ Pair<float> add2(Pair<float> x, Pair<float> y) {
  Pair<float> o;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(o.r) : "l"(x.r), "l"(y.r));
  return o;
}
template <> __device__ __forceinline__ Pair<float> mul2(Pair<float> x, Pair<float> y) {
  Pair<float> o;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o.r) : "l"(x.r), "l"(y.r));
  return o;
}
template <> __device__ __forceinline__ Pair<float> fma2(Pair<float> x, Pair<float> y,
                                                        Pair<float> z) {
  Pair<float> o;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(o.r) : "l"(x.r), "l"(y.r), "l"(z.r));
  return o;
}
// Two neighbouring elements widened, and rounded back.
template <class T> __device__ __forceinline__ Pair<acc_t<T>> widen2(const Vec<T, 2>& v) {
  return Pair<acc_t<T>>(load_acc<T>(v.v[0]), load_acc<T>(v.v[1]));
}
template <> __device__ __forceinline__ Pair<float> widen2(const Vec<__nv_bfloat16, 2>& v) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
  return Pair<float>(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <> __device__ __forceinline__ Pair<float> widen2(const Vec<__half, 2>& v) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return Pair<float>(f.x, f.y);
}
template <class T> __device__ __forceinline__ Vec<T, 2> narrow2(Pair<acc_t<T>> p) {
  return Vec<T, 2>{{round_to<T>(p.lo()), round_to<T>(p.hi())}};
}
template <> __device__ __forceinline__ Vec<__nv_bfloat16, 2> narrow2<__nv_bfloat16>(Pair<float> p) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(p.lo(), p.hi());
  return *reinterpret_cast<const Vec<__nv_bfloat16, 2>*>(&h);
}
template <> __device__ __forceinline__ Vec<__half, 2> narrow2<__half>(Pair<float> p) {
  const __half2 h = __floats2half2_rn(p.lo(), p.hi());
  return *reinterpret_cast<const Vec<__half, 2>*>(&h);
}

// ---- launches that overlap the kernel before them ---------------------------------
// Kernels of one call that follow each other: launched with
// programmatic stream serialisation, a kernel's blocks are set up while the one
// before is still running; after_previous(), before any access to memory, waits
// until that one has completed. Only for kernels whose predecessor in the
// stream is a kernel of the same call.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Lets the next kernel's blocks be set up from here on.
__device__ __forceinline__ void before_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <class... P, class... A>
stade_status launch_next(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                         A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  STADE_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
  count_launch();
  return STADE_OK;
}

inline bool known_dtype(int d) {
  return d == STADE_F32 || d == STADE_F64 || d == STADE_BF16 || d == STADE_F16;
}
inline size_t dtype_size(int d) { return d == STADE_F64 ? 8 : d == STADE_F32 ? 4 : 2; }

// Calls f with a value of the dtype's element type.
template <class F>
stade_status with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case STADE_F32: return f(float{});
    case STADE_F64: return f(double{});
    case STADE_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

// opts->flags of the reverse sweeps: whether adjoint outputs are added to (the
// generated convention) and whether the consumed seed is set to zero.
inline bool accumulates(const stade_opts* o) { return !(flags_of(o) & STADE_ADJ_STORE); }
inline bool consumes(const stade_opts* o) { return !(flags_of(o) & STADE_SEED_KEEP); }

// Largest power of two, at most 16 bytes, that divides every given address
// and the row length in bytes: what one vector access of a row may be.
inline int row_align(size_t row_bytes, std::initializer_list<const void*> ptrs) {
  uintptr_t m = row_bytes | 16u;
  for (const void* p : ptrs) m |= reinterpret_cast<uintptr_t>(p);
  return (int)(m & (~m + 1));
}

// a * b for sizes already known to be >= 0; false when it passes 2^62.
inline bool mul_ok(int64_t a, int64_t b, int64_t* out) {
  if (a != 0 && b > (int64_t(1) << 62) / a) return false;
  *out = a * b;
  return true;
}

}  // namespace stade
