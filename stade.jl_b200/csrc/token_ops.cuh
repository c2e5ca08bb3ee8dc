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
template <> __device__ __forceinline__ float load_acc(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float load_acc(__half v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T round_to(acc_t<T> v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements moved as one load or store (V * sizeof(T) = 2 .. 16
// bytes, the address a multiple of that).
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <class T, int V>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, acc_t<T> (&out)[V]) {
  const Vec<T, V> r = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = load_acc<T>(r.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const acc_t<T> (&in)[V]) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = round_to<T>(in[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = r;
}
template <class T, int V>
__device__ __forceinline__ void store_zero(T* __restrict__ p) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = round_to<T>(acc_t<T>(0));
  *reinterpret_cast<Vec<T, V>*>(p) = r;
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
