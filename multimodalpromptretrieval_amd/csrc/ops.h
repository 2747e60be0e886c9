// ops.h — what the tensor operators of ops.py (embed.hip, preference.hip, gradclip.hip, xattn.hip)
// share: the storage types and their conversions, reductions, the C entries' guard.
#pragma once

#include "common.h"

namespace mpr {

// Storage types (the dtype codes of mpr.h).  Arithmetic is fp32 or wider everywhere.
typedef __bf16 bf16;
typedef _Float16 f16;

// A run of N elements at element alignment: rows of odd length start anywhere, and gfx950's
// global loads and stores take any alignment of the element (one wide access, not N).
template <class T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T>
struct Vec<T, 1> {
  typedef T type;
};
template <class T>
constexpr int VEC16 = 16 / (int)sizeof(T);  // elements of one 16-byte access

template <class T>
__device__ __forceinline__ float to_f(T x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_f(float x) { return (T)x; }  // round to nearest even

template <class T, int N>
__device__ __forceinline__ float vec_f(const typename Vec<T, N>::type& v, int i) {
  if constexpr (N == 1) return to_f<T>(v);
  else return to_f<T>(v[i]);
}
template <class T, int N>
__device__ __forceinline__ void load_f(const T* p, float (&x)[N]) {
  const typename Vec<T, N>::type v = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = vec_f<T, N>(v, i);
}
template <class T, int N>
__device__ __forceinline__ void store_f(T* p, const float (&x)[N]) {
  typename Vec<T, N>::type v;
  if constexpr (N == 1) v = from_f<T>(x[0]);
  else
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_f<T>(x[i]);
  *reinterpret_cast<typename Vec<T, N>::type*>(p) = v;
}

// STREAM: past the caches, for results larger than they are.  Written the usual way, such a result
// leaves the 256 MB Infinity Cache full of lines that the next kernels' reads have to wait out:
// 262144 looked-up rows of 2 KB and the gradient after them 310 us, streamed 283.
template <class T, int N, bool STREAM>
__device__ __forceinline__ void store_f(T* p, const float (&x)[N]) {
  if constexpr (STREAM) {
    typename Vec<T, N>::type v;
    if constexpr (N == 1) v = from_f<T>(x[0]);
    else
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = from_f<T>(x[i]);
    __builtin_nontemporal_store(v, reinterpret_cast<typename Vec<T, N>::type*>(p));
  } else {
    store_f<T, N>(p, x);
  }
}
constexpr int64_t STREAM_BYTES = (int64_t)256 << 20;

template <class A>
__device__ __forceinline__ A wave_add(A v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Calls f(T{}) with the storage type of a dtype code that the entry has checked.
template <class F>
int by_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case MPR_F32: return f(float{});
    case MPR_BF16: return f(bf16{});
    case MPR_F16: return f(f16{});
  }
  set_error("dtype code %d (0 float32, 1 bfloat16, 2 float16)", (int)dtype);
  return MPR_EINVAL;
}

template <class F>
int ops_call(const char* what, F&& f) {
  try {
    return f();
  } catch (...) {
    set_error("%s: exception", what);
    return MPR_EINVAL;
  }
}
inline hipStream_t op_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

// A launch has less than 2^32 threads along x: blocks of up to 512 threads.
constexpr int64_t MAX_GRID_X = ((int64_t)1 << 23) - 1;

}  // namespace mpr
