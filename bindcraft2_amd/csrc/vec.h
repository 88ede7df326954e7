// Vectors of f32, binary16 or bfloat16 elements in memory, as f32 in registers.
#pragma once
#include "common.h"

namespace bc2n {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;

// A pointer read from a table does not tell the compiler that it is to global
// memory, and flat loads would wait on the LDS counter too.
template <class R>
__device__ __forceinline__ __attribute__((address_space(1))) R* global_ptr(const void* p) {
  return (__attribute__((address_space(1))) R*)(uintptr_t)p;
}

// 16 bytes of T, at any address aligned to one element (a global load or
// store of four dwords takes those on gfx950)
template <class T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    u32x4 v;
  };
  // ONCE: nontemporal, for what passes by once and would only displace what is
  // read again
  template <bool ONCE = false>
  static __device__ __forceinline__ u32x4 load(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(&global_ptr<const Raw>(p)->v);
    else return global_ptr<const Raw>(p)->v;
  }
  template <bool ONCE = false>
  static __device__ __forceinline__ void store(T* p, u32x4 v) {
    if constexpr (ONCE) __builtin_nontemporal_store(v, &global_ptr<Raw>(p)->v);
    else global_ptr<Raw>(p)->v = v;
  }
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) {
    typedef T Tv __attribute__((ext_vector_type(N)));
    const Tv h = __builtin_bit_cast(Tv, v);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)h[i];
  }
  // rounded to nearest even, once
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    typedef T Tv __attribute__((ext_vector_type(N)));
    Tv h;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = (T)x[i];
    return __builtin_bit_cast(u32x4, h);
  }
};

// N consecutive elements as f32, at any address aligned to one element
template <class T, int N>
struct Few {
  typedef T V __attribute__((ext_vector_type(N)));
  struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    V v;
  };
  template <bool ONCE>
  static __device__ __forceinline__ void load(const T* p, float* x) {
    V v;
    if constexpr (ONCE) v = __builtin_nontemporal_load(&global_ptr<const Raw>(p)->v);
    else v = global_ptr<const Raw>(p)->v;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  }
  // rounded to nearest even, once
  template <bool ONCE>
  static __device__ __forceinline__ void store(T* p, const float* x) {
    V v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    if constexpr (ONCE) __builtin_nontemporal_store(v, &global_ptr<Raw>(p)->v);
    else global_ptr<Raw>(p)->v = v;
  }
};

}  // namespace bc2n
