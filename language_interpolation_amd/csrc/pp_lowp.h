// 32- and 16-bit element types of the sequence-model operators (pp_recurrence.hip, pp_policy.hip,
// pp_adamw.hip): everything is computed in fp32, these helpers are the loads and stores around it.
// A store to 16 bits rounds to nearest even once, from the finished fp32 value.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __bf16 pp_bf16;
typedef _Float16 pp_f16;

template <typename T>
struct PPPair;  // two neighbouring elements in 32 bits (16-bit types)
template <>
struct PPPair<pp_bf16> {
  static __device__ __forceinline__ void get(uint32_t w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    typedef pp_bf16 v2 __attribute__((ext_vector_type(2)));
    v2 v;
    v.x = (pp_bf16)a;
    v.y = (pp_bf16)b;
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct PPPair<pp_f16> {
  static __device__ __forceinline__ void get(uint32_t w, float& a, float& b) {
    typedef pp_f16 v2 __attribute__((ext_vector_type(2)));
    const v2 v = __builtin_bit_cast(v2, w);
    a = (float)v.x;
    b = (float)v.y;
  }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    typedef pp_f16 v2 __attribute__((ext_vector_type(2)));
    v2 v;
    v.x = (pp_f16)a;
    v.y = (pp_f16)b;
    return __builtin_bit_cast(uint32_t, v);
  }
};

// N consecutive elements as raw 32-bit words, loaded and stored in one access (N * sizeof(T) = 2
// to 16 bytes, the address a multiple of that unless said otherwise), and their fp32 values.
template <int BYTES>
struct PPRaw;
template <>
struct PPRaw<2> { typedef uint16_t type; };
template <>
struct PPRaw<4> { typedef uint32_t type; };
template <>
struct PPRaw<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct PPRaw<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };

template <typename T, int N>
struct PPElems {
  typedef typename PPRaw<N * sizeof(T)>::type raw;
  static __device__ __forceinline__ raw load(const T* p) { return *reinterpret_cast<const raw*>(p); }
  static __device__ __forceinline__ void store(T* p, raw r) { *reinterpret_cast<raw*>(p) = r; }
  // at any element: one access all the same
  typedef raw loose __attribute__((aligned(sizeof(T))));
  static __device__ __forceinline__ raw load_any(const T* p) { return *reinterpret_cast<const loose*>(p); }
  static __device__ __forceinline__ void stream_any(T* p, raw r) {
    __builtin_nontemporal_store(r, reinterpret_cast<loose*>(p));
  }
  // what is read or written once: no place in the caches for it
  static __device__ __forceinline__ raw take(const T* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const raw*>(p));
  }
  static __device__ __forceinline__ void stream(T* p, raw r) {
    __builtin_nontemporal_store(r, reinterpret_cast<raw*>(p));
  }
  static __device__ __forceinline__ void get(const raw& r, float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
      struct S { float x[N]; };
      const S s = __builtin_bit_cast(S, r);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = s.x[i];
    } else if constexpr (N == 1) {
      v[0] = (float)__builtin_bit_cast(T, r);
    } else {
      struct S { uint32_t w[N / 2]; };
      const S s = __builtin_bit_cast(S, r);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) PPPair<T>::get(s.w[i], v[2 * i], v[2 * i + 1]);
    }
  }
  static __device__ __forceinline__ raw put(const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
      struct S { float x[N]; };
      S s;
#pragma unroll
      for (int i = 0; i < N; ++i) s.x[i] = v[i];
      return __builtin_bit_cast(raw, s);
    } else if constexpr (N == 1) {
      return __builtin_bit_cast(raw, (T)v[0]);
    } else {
      struct S { uint32_t w[N / 2]; };
      S s;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) s.w[i] = PPPair<T>::put(v[2 * i], v[2 * i + 1]);
      return __builtin_bit_cast(raw, s);
    }
  }
};
