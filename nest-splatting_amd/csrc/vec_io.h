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
    __builtin_memcpy(p, &t, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
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

}  // namespace nest
