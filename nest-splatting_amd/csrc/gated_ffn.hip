// Gated feed-forward block and its backward pass.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  y = h Wd^T
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// All products are summed in float32.  g and u are never stored by a forward
// pass alone; a training step keeps them in float32, because rounding them to
// 16 bits would make the gradients' error nearly twice one rounding.  h, dg
// and du are rounded to the inputs' type, as operands of the next product.
#include "blocks_internal.h"
#include "vec_io.h"

namespace nest {
namespace {

// ---- activations and their slopes ----

template <int kAct>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (kAct == NEST_ACT_RELU) return g <= 0.0f ? 0.0f : g;  // NaN stays
  if constexpr (kAct == NEST_ACT_SILU) return g / (1.0f + expf(-g));
  return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}

template <int kAct>
__device__ __forceinline__ float act_slope(float g) {
  if constexpr (kAct == NEST_ACT_RELU) return g > 0.0f ? 1.0f : 0.0f;
  if constexpr (kAct == NEST_ACT_SILU) {
    const float q = 1.0f / (1.0f + expf(-g));
    return q * (1.0f + g * (1.0f - q));
  }
  return 0.5f * (1.0f + erff(g * 0.70710678118654752f)) + g * expf(-0.5f * g * g) * 0.39894228040143268f;
}

// One product C = A B with element (m, k) of A at a[m am + k ak], (k, n) of B at
// b[n bn + k bk]; a second pair is added when given (dx sums two products).
template <typename T>
struct Product {
  const T *a, *b, *a2, *b2;
  int64_t am, ak, bn, bk;
  int64_t M, N, K;
};

constexpr int kSide = 64, kStep = 16;

template <typename T>
__device__ __forceinline__ void tile_product(const T* a, const T* b, const Product<T>& p, int64_t m0, int64_t n0,
                                             float (&acc)[4][4]) {
  __shared__ float as[kStep][kSide + 4], bs[kStep][kSide + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t k0 = 0; k0 < p.K; k0 += kStep) {
    __syncthreads();
    for (int t = threadIdx.x; t < kSide * kStep; t += 256) {
      // the index that is contiguous in memory runs over the lanes
      const int ka = p.ak == 1 ? t % kStep : t / kSide, ma = p.ak == 1 ? t / kStep : t % kSide;
      const int kb = p.bk == 1 ? t % kStep : t / kSide, nb = p.bk == 1 ? t / kStep : t % kSide;
      as[ka][ma] = m0 + ma < p.M && k0 + ka < p.K ? to_f32(a[(m0 + ma) * p.am + (k0 + ka) * p.ak]) : 0.0f;
      bs[kb][nb] = n0 + nb < p.N && k0 + kb < p.K ? to_f32(b[(n0 + nb) * p.bn + (k0 + kb) * p.bk]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(as[k][ty * 4 + i], bs[k][tx * 4 + j], acc[i][j]);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void product_kernel(Product<T> p, T* c) {
  const int64_t m0 = (int64_t)blockIdx.y * kSide, n0 = (int64_t)blockIdx.x * kSide;
  float acc[4][4] = {};
  tile_product(p.a, p.b, p, m0, n0, acc);
  if (p.a2) tile_product(p.a2, p.b2, p, m0, n0, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < p.M && n < p.N) c[m * p.N + n] = from_f32<T>(acc[i][j]);
    }
}

// g and u of a tile; h, and g and u where they are kept: kept[m][g 0..H, u 0..H].
template <typename T, int kAct>
__global__ __launch_bounds__(256) void gate_kernel(Product<T> p, T* h, float* kept) {
  const int64_t m0 = (int64_t)blockIdx.y * kSide, n0 = (int64_t)blockIdx.x * kSide;
  float g[4][4] = {}, u[4][4] = {};
  tile_product(p.a, p.b, p, m0, n0, g);
  tile_product(p.a, p.b2, p, m0, n0, u);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      if (h) h[m * p.N + n] = from_f32<T>(act_value<kAct>(g[i][j]) * u[i][j]);
      if (kept) {
        kept[m * 2 * p.N + n] = g[i][j];
        kept[m * 2 * p.N + p.N + n] = u[i][j];
      }
    }
}

// dh of a tile, turned into dg, du and h with the kept g and u.
template <typename T, int kAct>
__global__ __launch_bounds__(256) void gate_backward_kernel(Product<T> p, const float* kept, T* dg, T* du, T* h) {
  const int64_t m0 = (int64_t)blockIdx.y * kSide, n0 = (int64_t)blockIdx.x * kSide;
  float dh[4][4] = {};
  tile_product(p.a, p.b, p, m0, n0, dh);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      const float g = kept[m * 2 * p.N + n], u = kept[m * 2 * p.N + p.N + n], a = act_value<kAct>(g);
      dg[m * p.N + n] = from_f32<T>(dh[i][j] * u * act_slope<kAct>(g));
      du[m * p.N + n] = from_f32<T>(dh[i][j] * a);
      h[m * p.N + n] = from_f32<T>(a * u);
    }
}

template <typename T>
dim3 tiles(const Product<T>& p) {
  return dim3((unsigned)((p.N + kSide - 1) / kSide), (unsigned)((p.M + kSide - 1) / kSide));
}

template <typename T, int kAct>
hipError_t forward(const GatedParams& p, hipStream_t s) {
  const T *x = static_cast<const T*>(p.x), *wg = static_cast<const T*>(p.w_gate), *wu = static_cast<const T*>(p.w_up);
  const int64_t R = p.rows, I = p.in, H = p.hidden, O = p.out;
  T* h = static_cast<T*>(p.h);
  const Product<T> up{x, wg, nullptr, wu, I, 1, I, 1, R, H, I};
  gate_kernel<T, kAct><<<tiles(up), 256, 0, s>>>(up, h, p.kept);
  const Product<T> down{h, static_cast<const T*>(p.w_down), nullptr, nullptr, H, 1, H, 1, R, O, H};
  product_kernel<T><<<tiles(down), 256, 0, s>>>(down, static_cast<T*>(p.y));
  return hipGetLastError();
}

template <typename T, int kAct>
hipError_t backward(const GatedParams& p, hipStream_t s) {
  const T *x = static_cast<const T*>(p.x), *wg = static_cast<const T*>(p.w_gate), *wu = static_cast<const T*>(p.w_up),
          *wd = static_cast<const T*>(p.w_down), *dy = static_cast<const T*>(p.dy);
  const int64_t R = p.rows, I = p.in, H = p.hidden, O = p.out;
  T *h = static_cast<T*>(p.h), *dg = static_cast<T*>(p.dg), *du = static_cast<T*>(p.du);
  if (R > 0) {
    if (p.kept_here) {
      const Product<T> up{x, wg, nullptr, wu, I, 1, I, 1, R, H, I};
      gate_kernel<T, kAct><<<tiles(up), 256, 0, s>>>(up, nullptr, p.kept);
    }
    const Product<T> dh{dy, wd, nullptr, nullptr, O, 1, 1, H, R, H, O};
    gate_backward_kernel<T, kAct><<<tiles(dh), 256, 0, s>>>(dh, p.kept, dg, du, h);
    if (p.dx) {
      const Product<T> q{dg, wg, du, wu, H, 1, 1, I, R, I, H};
      product_kernel<T><<<tiles(q), 256, 0, s>>>(q, static_cast<T*>(p.dx));
    }
  }
  if (p.dw_gate) {
    const Product<T> q{dg, x, nullptr, nullptr, 1, H, 1, I, H, I, R};
    product_kernel<T><<<tiles(q), 256, 0, s>>>(q, static_cast<T*>(p.dw_gate));
  }
  if (p.dw_up) {
    const Product<T> q{du, x, nullptr, nullptr, 1, H, 1, I, H, I, R};
    product_kernel<T><<<tiles(q), 256, 0, s>>>(q, static_cast<T*>(p.dw_up));
  }
  if (p.dw_down) {
    const Product<T> q{dy, h, nullptr, nullptr, 1, O, 1, H, O, H, R};
    product_kernel<T><<<tiles(q), 256, 0, s>>>(q, static_cast<T*>(p.dw_down));
  }
  return hipGetLastError();
}

template <typename T>
hipError_t run(const GatedParams& p, hipStream_t s, bool back) {
  if (p.activation == NEST_ACT_RELU) return back ? backward<T, NEST_ACT_RELU>(p, s) : forward<T, NEST_ACT_RELU>(p, s);
  if (p.activation == NEST_ACT_SILU) return back ? backward<T, NEST_ACT_SILU>(p, s) : forward<T, NEST_ACT_SILU>(p, s);
  return back ? backward<T, NEST_ACT_GELU>(p, s) : forward<T, NEST_ACT_GELU>(p, s);
}

}  // namespace

hipError_t launch_gated_ffn(const GatedParams& p, hipStream_t s, bool back) {
  if (p.dtype == NEST_DTYPE_F32) return run<float>(p, s, back);
  return p.dtype == NEST_DTYPE_F16 ? run<f16_t>(p, s, back) : run<bf16_t>(p, s, back);
}

}  // namespace nest
