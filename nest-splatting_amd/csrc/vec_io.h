// Vectors of one element type in memory and float32 in registers, for the
// row-wise operators (layer_norm.hip, dropout.hip, gated_ffn.hip).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nest {

// 16 bytes of T; kept as bytes that need no more than T's own alignment, so
// that rows of odd length load with the same wide instructions (gfx950 loads
// and stores unaligned dwordx4).
template <typename T>
struct Vec16 {
  static constexpr int kN = 16 / (int)sizeof(T);
  T v[kN];
};

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

// Nearest even, as every store of a 16-bit result here.
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// n valid elements at p (n may be <= 0 or above kN): the rest read as zero.
template <typename T>
__device__ __forceinline__ Vec16<T> load_raw(const T* p, int n) {
  constexpr int N = Vec16<T>::kN;
  Vec16<T> t;
  if (n >= N) {
    __builtin_memcpy(&t, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) t.v[i] = i < n ? p[i] : (T)0.0f;
  }
  return t;
}

// 4, 8 or 16 bytes at any alignment, as one store: of elements the compiler
// would share the last ones with the code of a shorter row's end, and split the
// rest (three requests a store instead of one).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
template <typename V>
__device__ __forceinline__ void store_whole(void* p, const V& v) {
  if constexpr (sizeof(V) == 16) *static_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4_any, v);
  else if constexpr (sizeof(V) == 8) *static_cast<u32x2_any*>(p) = __builtin_bit_cast(u32x2_any, v);
  else *static_cast<u32_any*>(p) = __builtin_bit_cast(uint32_t, v);
}

// The same 16 bytes as words: where a load may be skipped, an array of 16-bit
// elements takes a register each from there to its use, twice as many.
template <typename T>
struct Words16 {
  static constexpr int kN = 16 / (int)sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ T operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, w[i]);
    else return __builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (i % 2 * 16)));
  }
};

// kWhole: rows are whole vectors, so n is <= 0 or kN at least.
template <bool kWhole, typename T>
__device__ __forceinline__ Words16<T> load_words(const T* p, int n) {
  constexpr int N = Words16<T>::kN;
  Words16<T> t = {{0, 0, 0, 0}};
  if (kWhole ? n > 0 : n >= N) {
    __builtin_memcpy(&t, p, 16);
  } else if (!kWhole) {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) {
        if constexpr (sizeof(T) == 4) t.w[i] = __builtin_bit_cast(uint32_t, p[i]);
        else t.w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (i % 2 * 16);
      }
  }
  return t;
}

template <typename T>
__device__ __forceinline__ void load_vec(float (&f)[Vec16<T>::kN], const T* p, int n) {
  const Vec16<T> t = load_raw(p, n);
#pragma unroll
  for (int i = 0; i < Vec16<T>::kN; i++) f[i] = to_f32(t.v[i]);
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[Vec16<T>::kN], int n) {
  constexpr int N = Vec16<T>::kN;
  if (n >= N) {
    Vec16<T> t;
#pragma unroll
    for (int i = 0; i < N; i++) t.v[i] = from_f32<T>(f[i]);
    store_whole(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
}

// The first n of a vector's elements (n may be <= 0 or above kN).
template <typename T>
__device__ __forceinline__ void store_raw(T* p, const Vec16<T>& t, int n) {
  constexpr int N = Vec16<T>::kN;
  if (n >= N) {
    store_whole(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) p[i] = t.v[i];
  }
}

template <bool kWhole, typename T>
__device__ __forceinline__ void store_piece(T* p, const Vec16<T>& t, int n) {
  if constexpr (!kWhole) store_raw(p, t, n);
  else if (n > 0) store_whole(p, t);
}

// N parameters (weights, biases) of a type of their own as float32.
template <typename P, int N>
__device__ __forceinline__ void load_param(float (&f)[N], const P* p, int n) {
  constexpr int K = Vec16<P>::kN;
  if constexpr (K <= N) {
#pragma unroll
    for (int v = 0; v < N / K; v++) {
      const Vec16<P> t = load_raw(p + v * K, n - v * K);
#pragma unroll
      for (int i = 0; i < K; i++) f[v * K + i] = to_f32(t.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

// The first n of N values as parameters of a type of their own.
template <typename P, int N>
__device__ __forceinline__ void store_param(P* p, const float (&f)[N], int n) {
  constexpr int K = Vec16<P>::kN;
  static_assert(N % K == 0, "");
#pragma unroll
  for (int v = 0; v < N / K; v++) {
    Vec16<P> t;
#pragma unroll
    for (int i = 0; i < K; i++) t.v[i] = from_f32<P>(f[v * K + i]);
    store_raw(p + v * K, t, n - v * K);
  }
}

}  // namespace nest
