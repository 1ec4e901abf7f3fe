// Element types of the operators on invariant features (embedding, attention, gated feed-forward): storage types, the
// type sums are held in, and loads and stores of V consecutive elements as one transaction.
#pragma once

#include "cgtp_device.h"
#include "cgtp_host.h"

namespace cgtp {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };

template <typename T, int V> struct ElemVec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct ElemVec<T, 1> { typedef T type; };

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

// Vectors at an address aligned to an element only: the hardware reads and writes such by itself.  Their type is an integer
// vector on purpose: taken as elements, the compiler splits the access.
template <typename T, typename R> struct LooseOf { typedef R type __attribute__((aligned(sizeof(T)))); };

// V elements, 16 bytes of them or one, widened to the accumulation type.
template <typename T, int V, typename A>
__device__ __forceinline__ void load_elems(A (&dst)[V], const T* p) {
  if constexpr (V == 1) {
    dst[0] = (A)p[0];
  } else {
    static_assert(V * sizeof(T) == 16);
    const typename ElemVec<T, V>::type v = __builtin_bit_cast(typename ElemVec<T, V>::type, *reinterpret_cast<const typename LooseOf<T, u32x4_t>::type*>(p));
#pragma unroll
    for (int i = 0; i < V; ++i) dst[i] = (A)v[i];
  }
}
// STREAM: past the caches' keep: what is written once should not displace what is read again.
template <typename T, int V, bool STREAM = false, typename A>
__device__ __forceinline__ void store_elems(T* p, const A (&src)[V]) {
  if constexpr (V == 1) {
    p[0] = (T)src[0];
  } else {
    typename ElemVec<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)src[i];
    const u32x4_t r = __builtin_bit_cast(u32x4_t, v);
    if constexpr (STREAM) __builtin_nontemporal_store(r, reinterpret_cast<typename LooseOf<T, u32x4_t>::type*>(p));
    else *reinterpret_cast<typename LooseOf<T, u32x4_t>::type*>(p) = r;
  }
}

// N = sizeof(R) / sizeof(T) elements, the ones from `valid` (at least 1) on as zeros.  Only a vector that crosses the end is
// taken apart.
template <typename R, typename T>
__device__ __forceinline__ R load_part(const T* p, int64_t valid) {
  constexpr int N = sizeof(R) / sizeof(T);
  if (valid >= N) return *reinterpret_cast<const typename LooseOf<T, R>::type*>(p);
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const T v = p[i < valid ? i : 0];
    e[i] = i < valid ? v : T(0);
  }
  R r;
  __builtin_memcpy(&r, e, sizeof(R));
  return r;
}
// The first `valid` of N elements.
template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const T (&e)[N], int64_t valid) {
  typedef unsigned raw_t __attribute__((ext_vector_type(N * sizeof(T) / 4)));
  if (valid >= N) {
    raw_t r;
    __builtin_memcpy(&r, e, sizeof(r));
    *reinterpret_cast<typename LooseOf<T, raw_t>::type*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) p[i] = e[i];
  }
}

// Eight values rounded to an element-aligned address, the first `valid` of them.
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&src)[8], int64_t valid) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += N) {
    if (valid <= i) continue;
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)src[i + j];
    store_part<T, N>(p + i, v, valid - i);
  }
}

// acc + a b with 32 x 32 results: a pair of chunks of 16 bytes along k, one for each half of the wavefront.
template <typename T>
__device__ __forceinline__ f32x16_t mma_pair(const u32x4_t& a, const u32x4_t& b, f32x16_t acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[j], fb[j], acc, 0, 0, 0);
  } else if constexpr (__is_same(T, f16_t)) {
    typedef f16_t v8 __attribute__((ext_vector_type(8)));
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  } else {
    typedef bf16_t v8 __attribute__((ext_vector_type(8)));
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  }
  return acc;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? CGTP_OK : CGTP_ERR_LAUNCH; }

}  // namespace cgtp
