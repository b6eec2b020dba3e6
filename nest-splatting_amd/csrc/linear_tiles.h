// A dense layer for one element type, in tiles.
//
//   z = x W^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// The products run in the tiles of tile_gemm.h, few rows as in gated_few.h.
// The forward's epilogue takes the float32 sums through LDS, so that a lane
// has 16 bytes of a row: it adds the bias, applies the activation, adds the
// residual and rounds once.  A training call keeps the slopes act'(z) there,
// since they lie in [-0.13, 1.13] and a fixed point of 16 bits (steps of
// 1/26000: 2^-15.7 off at most) loses nothing beside a 16-bit dz; z itself in
// 16 bits would make the gradients' error 1.7 times one rounding instead of
// 1.4, and in float32 cost twice the bytes.  float32 keeps float32 slopes.  In
// 8 bits (steps of 1/200, 0 and 1 among them, 2^-8.6 off at most: about what a
// bfloat16 rounding of z makes) they take one byte, for 16-bit types; float32
// then takes 16 bits.  ReLU's slopes, 0 and 1, always take one byte.
//
// The backward makes dz, rounded to the type as the next products' operand, in
// one pass that also gathers db from the unrounded values.
//
// 8192 rows of 2048 -> 8192 bf16 with GELU: forward 318 us (865 TFLOP/s; the
// epilogue's exponentials and 268 MB of y and slopes stand behind the matrix
// cores, 0.45 busy), dx 237 and dW 232 (1160 and 1185 TFLOP/s, 0.65 busy; the
// library's 8192^3 product reaches 1380, its second operand transposed 1577), dz
// 77 (402 MB: 5.2 TB/s).
#pragma once

#include "column_sums.h"
#include "gated_few.h"
#include "gated_tiles.h"
#include "residual_internal.h"

namespace nest {
namespace {

// ---- activations and kept slopes ----

template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  if (act == NEST_ACT_NONE) f(ActConstant<NEST_ACT_NONE>());
  else with_act(act, f);
}

// GELU of a 16-bit result: Phi(-|z|) = exp(-z^2 / 2) t P(t) with t = 1 / (1 +
// 0.3 |z|), so that it keeps its relative accuracy however small it gets, and a
// result its one rounding.  P, of degree 5, was fitted to erfcx(|z| / sqrt(2)) /
// (2 t) over |z| <= 14 by minimising the largest error beside 1e-6 + 1.2e-7 /
// Phi(-|z|), at most 1.6e-5: it is off by 1.3e-5 of Phi at most, below |z| = 1 by
// 1.3e-6.  The exponential serves the slope's density too: 16 operations and
// two for the slope (the narrow forward is bound by them).
template <typename T, int kAct, bool kSlope = true>
__device__ __forceinline__ float activate(float z, float& slope) {
  if constexpr (kAct == NEST_ACT_NONE) {
    slope = 1.0f;
    return z;
  } else if constexpr (kAct == NEST_ACT_GELU && sizeof(T) == 2) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(z), 1.0f));
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
    const float tail = t * e *
        fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.0797698168f, 0.223536754f), -0.0248124557f), 0.14800684f), 0.112895661f), 0.120143082f);
    const float phi = z < 0.0f ? tail : 1.0f - tail;
    if constexpr (kSlope) slope = fmaf(z * e, 0.39894228040143268f, phi);
    return z * phi;
  } else {
    return act_value<T, kAct, kSlope>(z, slope);
  }
}

constexpr float kFine = 26000.0f, kCoarse = 200.0f;
constexpr int kCoarseZero = 26;             // the code of a slope of 0

__device__ __forceinline__ int16_t fine_code(float s) { return s == s ? (int16_t)__builtin_rintf(s * kFine) : (int16_t)-32768; }
__device__ __forceinline__ uint8_t coarse_code(float s) {
  return s == s ? (uint8_t)(__builtin_rintf(s * kCoarse) + (float)kCoarseZero) : (uint8_t)255;
}
__device__ __forceinline__ float slope_of(int16_t c) { return c == -32768 ? __builtin_nanf("") : (float)c * (1.0f / kFine); }
// of a byte's value
__device__ __forceinline__ float coarse_slope(float c) { return c == 255.0f ? __builtin_nanf("") : (c - (float)kCoarseZero) * (1.0f / kCoarse); }
__device__ __forceinline__ float slope_of(uint8_t c) { return coarse_slope((float)c); }
__device__ __forceinline__ float slope_of(float c) { return c; }

// n of K elements of a type of any size at p, with no more than its alignment.
template <typename E, int K>
struct Pack {
  E v[K];
  __device__ __forceinline__ void store(E* p, int n) const {
    if (n >= K) {
      store_whole(p, *this);
    } else {
#pragma unroll
      for (int i = 0; i < K; i++)
        if (i < n) p[i] = v[i];
    }
  }
  __device__ __forceinline__ void load(const E* p, int n) {
    if (n >= K) {
      __builtin_memcpy(v, p, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < K; i++) v[i] = i < n ? p[i] : (E)0;
    }
  }
};

// ---- the forward's epilogue ----

template <typename T>
struct Epilogue {
  const T *bias, *residual;
  T* y;
  void* kept;
  int slope_bytes, act, N;

  // K sums of a row from column c on, n of them inside.
  template <int K, int kAct>
  __device__ __forceinline__ void finish(int64_t row, int c, int n, float (&z)[K]) const {
    const int64_t at = row * N + c;
    if (bias) {
      float b[K];
      load_param(b, bias + c, n);
#pragma unroll
      for (int i = 0; i < K; i++) z[i] += b[i];
    }
    float slope[K];
#pragma unroll
    for (int i = 0; i < K; i++) z[i] = activate<T, kAct>(z[i], slope[i]);
    if (kAct != NEST_ACT_NONE && kept) {
      if (slope_bytes == 1) {
        Pack<uint8_t, K> s;
#pragma unroll
        for (int i = 0; i < K; i++) s.v[i] = coarse_code(slope[i]);
        s.store(static_cast<uint8_t*>(kept) + at, n);
      } else if (slope_bytes == 2) {
        Pack<int16_t, K> s;
#pragma unroll
        for (int i = 0; i < K; i++) s.v[i] = fine_code(slope[i]);
        s.store(static_cast<int16_t*>(kept) + at, n);
      } else if constexpr (sizeof(T) == 4) {
        Pack<float, K> s;
#pragma unroll
        for (int i = 0; i < K; i++) s.v[i] = slope[i];
        s.store(static_cast<float*>(kept) + at, n);
      }
    }
    if (residual) {
      float r[K];
      load_param(r, residual + at, n);
#pragma unroll
      for (int i = 0; i < K; i++) z[i] += r[i];
    }
    store_param(y + at, z, n);
  }
};

template <typename T>
struct LinearTiles {
  const T *x, *w;      // [M][ldx], [N][ldx]
  int64_t ldx;
  int M, N;
  Epilogue<T> ep;
  int tiles_m, tiles_n, splits;
  float* part;         // [splits][M][N], or null where splits is 1
};

// 16 rows of a wave's sums, row by row.
template <int FN>
struct SumStage {
  static constexpr int kPitch = FN * 16 + 4;
  float v[16 * kPitch];
};

template <typename T, typename C>
__global__ __launch_bounds__(C::NT) void linear_tile_kernel(LinearTiles<T> p) {
  const int split = p.splits > 1 ? blockIdx.x % p.splits : 0;
  int tm, tn;
  tile_of(p.splits > 1 ? blockIdx.x / p.splits : blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  constexpr int kStep = kStepBytes / (int)sizeof(T), K = Vec16<T>::kN;
  const int64_t per = ((p.ldx + kStep - 1) / kStep + p.splits - 1) / p.splits * kStep;
  const int64_t k0 = split * per, k = p.ldx - k0 < per ? p.ldx - k0 : per;
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
  f32x4 acc[C::FM][C::FN] = {};
  Loader<T, true, C::BM, C::NT> la;
  Loader<T, true, C::BN, C::NT> lb;
  la.init(p.x + k0, p.ldx, m0, p.M);
  lb.init(p.w + k0, p.ldx, n0, p.N);
  tile_product<T, true, true, C>(la, lb, k, nullptr, nullptr, acc);   // a split past the end has k <= 0: it loads zeros
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // made again here, not held in a register over the products
  const int w = wave_id();
  const int64_t m = m0 + (w / C::WN) * C::FM * 16;
  const int n = (int)n0 + (w % C::WN) * C::FN * 16;
  if (p.part) {
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < C::FM; i++) {
      if (m + i * 16 + r >= p.M) continue;
#pragma unroll
      for (int j = 0; j < C::FN; j++)
        store4(p.part + (split * (int64_t)p.M + m + i * 16 + r) * p.N, n + j * 16 + q * 4, p.N, p.N % 4 == 0, acc[i][j]);
    }
    return;
  }
  __syncthreads();   // the operands' LDS is free
  typedef SumStage<C::FN> Stage;
  static_assert(sizeof(Stage) * (C::NT / 64) <= (C::BM + C::BN) * kStepBytes, "");
  Stage& stage = reinterpret_cast<Stage*>(tile_lds<C>())[w];
  constexpr int kRow = C::FN * 16 / K;   // pieces of a row
  with_activation(p.ep.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < C::FM; i++) {
#pragma unroll
      for (int j = 0; j < C::FN; j++)
        *reinterpret_cast<f32x4*>(&stage.v[(lane & 15) * Stage::kPitch + j * 16 + (lane >> 4) * 4]) = acc[i][j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int u = 0; u < 16 * kRow / 64; u++) {
        const int t = u * 64 + lane, r = t / kRow, c = (t % kRow) * K;
        const int64_t row = m + i * 16 + r;
        float v[K];
#pragma unroll
        for (int e = 0; e < K; e += 4) {
          const f32x4 s = *reinterpret_cast<const f32x4*>(&stage.v[r * Stage::kPitch + c + e]);
#pragma unroll
          for (int f = 0; f < 4; f++) v[e + f] = s[f];
        }
        if (row < p.M && n + c < p.N) p.ep.template finish<K, act.value>(row, n + c, p.N - n - c, v);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  });
}

// Joins the partial sums in the order of the splits, 16 bytes of y a thread.
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearTiles<T> p) {
  constexpr int K = Vec16<T>::kN;
  const int pieces = (p.N + K - 1) / K;
  const int64_t total = (int64_t)p.M * pieces, slice = (int64_t)p.M * p.N;
  with_activation(p.ep.act, [&](auto act) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
      const int64_t row = i / pieces;
      const int c = (int)(i - row * pieces) * K, n = p.N - c;
      float z[K] = {};
      for (int s = 0; s < p.splits; s += 2) {   // a power of two, two at least
        float a[K], b[K];
        load_param(a, p.part + s * slice + row * p.N + c, n);
        load_param(b, p.part + (s + 1) * slice + row * p.N + c, n);
#pragma unroll
        for (int e = 0; e < K; e++) z[e] = z[e] + a[e] + b[e];
      }
      p.ep.template finish<K, act.value>(row, c, n, z);
    }
  });
}

// The few-row kernel's sums, one by one.
template <typename T>
struct FinishSum {
  Epilogue<T> ep;
  __device__ __forceinline__ void operator()(const Few<T>& p, int row, int64_t c, float v) const {
    with_activation(ep.act, [&](auto act) {
      const int64_t at = (int64_t)row * ep.N + c;
      float slope;
      v = activate<T, act.value>(ep.bias ? v + to_f32(ep.bias[c]) : v, slope);
      if (act.value != NEST_ACT_NONE && ep.kept) {
        if (ep.slope_bytes == 1) static_cast<uint8_t*>(ep.kept)[at] = coarse_code(slope);
        else if (sizeof(T) == 2 || ep.slope_bytes == 2) static_cast<int16_t*>(ep.kept)[at] = fine_code(slope);
        else static_cast<float*>(ep.kept)[at] = slope;
      }
      ep.y[at] = from_f32<T>(ep.residual ? v + to_f32(ep.residual[at]) : v);
    });
  }
};

// ---- dz and db ----

template <typename T>
struct SlopeRows {
  const T* dy;         // [rows][N]
  const void* kept;    // [rows][N], or null: dz is dy
  int slope_bytes;
  int64_t rows;
  int N;
  int64_t ldz;
  T* dz;               // [rows][ldz], its pad columns zeros; or null
  float* part;         // [gridDim.y][N] sums of dz, or null
};

// A lane keeps K columns over its rows: 256 / lanes rows at a time.
template <typename T, typename E>
__global__ __launch_bounds__(256) void linear_slope_kernel(SlopeRows<T> p, int lanes) {
  constexpr int K = Vec16<T>::kN, U = 4;
  __shared__ float gather[256][K + 1];
  const int lane = threadIdx.x & (lanes - 1), sub = threadIdx.x / lanes, rows_wg = 256 / lanes;
  const int c = (blockIdx.x * lanes + lane) * K, n = p.N - c;
  float sum[K] = {};
  const int64_t step = (int64_t)gridDim.y * rows_wg;
  for (int64_t row = (int64_t)blockIdx.y * rows_wg + sub; row < p.rows; row += step * U) {
    Words16<T> d[U];
    Pack<E, K> s[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t r = row + u * step;
      d[u] = load_words<false>(p.dy + r * p.N + c, r < p.rows ? n : 0);
      if (p.kept) s[u].load(static_cast<const E*>(p.kept) + r * p.N + c, r < p.rows ? n : 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t r = row + u * step;
      float v[K];
#pragma unroll
      for (int i = 0; i < K; i++) {
        v[i] = to_f32(d[u][i]);
        if (p.kept) v[i] *= slope_of(s[u].v[i]);
        if (i >= n || r >= p.rows) v[i] = 0.0f;
        sum[i] += v[i];
      }
      if (p.dz && r < p.rows) store_vec<T>(p.dz + r * p.ldz + c, v, (int)(p.ldz - c));
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < K; i++) gather[threadIdx.x][i] = sum[i];
  __syncthreads();
  for (int t = threadIdx.x; t < lanes * K; t += 256) {
    float s = 0.0f;
    for (int r = 0; r < rows_wg; r++) s += gather[r * lanes + t / K][t % K];
    const int col = blockIdx.x * lanes * K + t;
    if (col < p.N) p.part[(int64_t)blockIdx.y * p.N + col] = s;
  }
}

template <typename T>
hipError_t launch_slopes(const SlopeRows<T>& p, int groups, hipStream_t s) {
  constexpr int K = Vec16<T>::kN;
  const int vecs = (int)((p.ldz + K - 1) / K);
  int lanes = 1;
  while (lanes < vecs && lanes < 64) lanes *= 2;
  const dim3 grid((unsigned)((vecs + lanes - 1) / lanes), (unsigned)groups);
  if (p.slope_bytes <= 1) linear_slope_kernel<T, uint8_t><<<grid, 256, 0, s>>>(p, lanes);
  else if (sizeof(T) == 2 || p.slope_bytes == 2) linear_slope_kernel<T, int16_t><<<grid, 256, 0, s>>>(p, lanes);
  else if constexpr (sizeof(T) == 4) linear_slope_kernel<T, float><<<grid, 256, 0, s>>>(p, lanes);
  return hipGetLastError();
}

}  // namespace
}  // namespace nest
