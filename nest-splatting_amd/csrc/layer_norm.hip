// Layer norm of each row and its backward pass.
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   y = (x - mean) rstd w + b
//   with g = dy w and h = (x - mean) rstd:
//   dx = rstd (g - sum g / D - h sum (g h) / D),  dw = sum_rows dy h,  db = sum_rows dy
//
// Memory bound: forward reads x and writes y, backward reads x and dy and
// writes dx.  A row is held in registers between its statistics and its
// output, so each array crosses HBM once; the variance is taken about the
// mean (a second pass over registers), never as a difference of squares.  All
// sums are float32; y, dx, dw and db are rounded once.
//
// A row of up to 192 vectors of 16 bytes belongs to a group of 1 to 64 lanes
// (several rows a wave for narrow rows), a longer one to a workgroup; past
// the registers of a workgroup the row is read again for each pass.  A group
// strides over its rows with the weights in registers and the next row on its
// way.
//
// Measured: 1,702,400 x 64 bf16 forward 83 us (5.3 TB/s), backward 136 us
// (4.8); 8192 x 4096 float32 55 us (4.9) and 80 us (5.0); 50,000 x 1155 f16,
// rows at odd addresses, 68 us (3.4) and 145 us (2.4: two waves a SIMD fit).
#include "blocks_internal.h"
#include "vec_io.h"

#include <type_traits>

namespace nest {
namespace {

constexpr int kLnThreads = 256;      // of rows that stay with a wave, and of the long kernels
constexpr int kLnMost = 1024;        // of rows a workgroup shares (512 for 16-bit rows: their lanes hold twice the values)
constexpr int kLnWaves = kLnMost / 64;
template <typename T>
constexpr int most_threads() { return sizeof(T) == 4 ? kLnMost : kLnMost / 2; }
constexpr int64_t kLnForwardGrid = 2048;   // workgroups

// Sums over the lanes of one row; every lane gets the result.
template <bool kBlock>
__device__ __forceinline__ float row_sum(float v, int lanes, float* lds) {
  if constexpr (kBlock) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < (int)blockDim.x / 64; w++) v += lds[w];
  } else {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  }
  return v;
}

template <typename T, typename P, int NV, bool kBlock>
__global__ __launch_bounds__(kBlock ? most_threads<T>() : kLnThreads) void layer_norm_kernel(LayerNormParams p, int lanes) {
  constexpr int N = Vec16<T>::kN;
  __shared__ float lds[2][kLnWaves];
  const int rows_wg = kBlock ? 1 : kLnThreads / lanes;
  const int lane = kBlock ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int D = p.cols;
  const float inv = 1.0f / (float)D;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  int64_t row = (int64_t)blockIdx.x * rows_wg + (kBlock ? 0 : threadIdx.x / lanes);
  Vec16<T> next[NV];
  auto load = [&](int64_t at) {
    const T* x = static_cast<const T*>(p.x) + at * D;
#pragma unroll
    for (int k = 0; k < NV; k++) next[k] = load_raw(x + (k * lanes + lane) * N, at < p.rows ? D - (k * lanes + lane) * N : 0);
  };
  load(row);
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int c = (k * lanes + lane) * N;
    load_param(w[k], static_cast<const P*>(p.weight) + c, D - c);
    load_param(b[k], static_cast<const P*>(p.bias) + c, p.bias ? D - c : 0);
  }
  for (; row < p.rows; row += step) {   // in kBlock the same number of turns for all threads
    float v[NV][N];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        v[k][i] = to_f32(next[k].v[i]);
        s += v[k][i];
      }
    load(row + step);   // on its way while this row is worked on
    const float mean = row_sum<kBlock>(s, lanes, lds[0]) * inv;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; i++) {
        v[k][i] -= mean;
        if (c + i < D) q = fmaf(v[k][i], v[k][i], q);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<kBlock>(q, lanes, lds[1]) * inv + p.eps);
    T* y = static_cast<T*>(p.y) + row * D;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; i++) v[k][i] = fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
      store_vec<T>(y + c, v[k], D - c);
    }
    if (lane == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
  }
}

// Rows past a workgroup's registers: three passes, the later two from cache.
template <typename T, typename P>
__global__ __launch_bounds__(kLnThreads) void layer_norm_long_kernel(LayerNormParams p) {
  constexpr int N = Vec16<T>::kN;
  __shared__ float lds[2][kLnWaves];
  const int D = p.cols;
  const float inv = 1.0f / (float)D;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
  const T* x = static_cast<const T*>(p.x) + row * D;
  T* y = static_cast<T*>(p.y) + row * D;
  float s = 0.0f, v[N];
  for (int c = threadIdx.x * N; c < D; c += kLnThreads * N) {
    load_vec<T>(v, x + c, D - c);
#pragma unroll
    for (int i = 0; i < N; i++) s += v[i];
  }
  const float mean = row_sum<true>(s, kLnThreads, lds[0]) * inv;
  float q = 0.0f;
  for (int c = threadIdx.x * N; c < D; c += kLnThreads * N) {
    load_vec<T>(v, x + c, D - c);
#pragma unroll
    for (int i = 0; i < N; i++)
      if (c + i < D) q = fmaf(v[i] - mean, v[i] - mean, q);
  }
  const float rstd = 1.0f / sqrtf(row_sum<true>(q, kLnThreads, lds[1]) * inv + p.eps);
  for (int c = threadIdx.x * N; c < D; c += kLnThreads * N) {
    float w[N], b[N];
    load_vec<T>(v, x + c, D - c);
    load_param(w, static_cast<const P*>(p.weight) + c, D - c);
    if (p.bias) load_param(b, static_cast<const P*>(p.bias) + c, D - c);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float h = (v[i] - mean) * rstd;
      v[i] = p.bias ? fmaf(h, w[i], b[i]) : h * w[i];
    }
    store_vec<T>(y + c, v, D - c);
  }
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  }
}

// Both sums of a row's backward at once; the LDS alternates between rows, so
// one barrier a row is enough.
template <bool kBlock>
__device__ __forceinline__ void row_sum2(float& a, float& b, int lanes, float (*lds)[kLnWaves]) {
  if constexpr (kBlock) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      a += __shfl_xor(a, o);
      b += __shfl_xor(b, o);
    }
    if ((threadIdx.x & 63) == 0) {
      lds[0][threadIdx.x >> 6] = a;
      lds[1][threadIdx.x >> 6] = b;
    }
    __syncthreads();
    a = b = 0.0f;
    for (int w = 0; w < (int)blockDim.x / 64; w++) {
      a += lds[0][w];
      b += lds[1][w];
    }
  } else {
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      a += __shfl_xor(a, o);
      b += __shfl_xor(b, o);
    }
  }
}

// Rows are dealt over the workgroups; a lane keeps the same columns for all
// of its rows, so dw and db gather in registers and each workgroup writes one
// row of partial sums: part[workgroup][dw, db][D].  The sums' order depends on
// the launch shape alone, so results repeat bit for bit.
template <typename T, typename P, int NV, bool kBlock>
__global__ __launch_bounds__(kBlock ? most_threads<T>() : kLnThreads) void layer_norm_backward_kernel(LayerNormParams p, int lanes) {
  constexpr int N = Vec16<T>::kN;
  __shared__ float lds[2][2][kLnWaves];
  __shared__ float gather[kBlock ? 1 : kLnThreads][N + 1];
  const int D = p.cols;
  const int rows_wg = kBlock ? 1 : kLnThreads / lanes;
  const int lane = kBlock ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int sub = kBlock ? 0 : threadIdx.x / lanes;
  const float inv = 1.0f / (float)D;
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int c = (k * lanes + lane) * N;
    load_param(w[k], static_cast<const P*>(p.weight) + c, D - c);
#pragma unroll
    for (int i = 0; i < N; i++) dw[k][i] = db[k][i] = 0.0f;
  }
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  int64_t row = (int64_t)blockIdx.x * rows_wg + sub;
  Vec16<T> nx[NV], ny[NV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto load = [&](int64_t at) {
    const bool in = at < p.rows;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N;
      nx[k] = load_raw(static_cast<const T*>(p.x) + at * D + c, in ? D - c : 0);
      ny[k] = load_raw(static_cast<const T*>(p.dy) + at * D + c, in ? D - c : 0);
    }
    if (in) {
      next_mean = p.mean[at];
      next_rstd = p.rstd[at];
    }
  };
  load(row);
  for (; row < p.rows; row += step, turn ^= 1) {
    float h[NV][N], g[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        h[k][i] = to_f32(nx[k].v[i]);
        g[k][i] = to_f32(ny[k].v[i]);
      }
    const float mean = next_mean, rstd = next_rstd;
    load(row + step);   // on its way while this row is worked on
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        h[k][i] = (h[k][i] - mean) * rstd;
        dw[k][i] = fmaf(g[k][i], h[k][i], dw[k][i]);
        db[k][i] += g[k][i];
        g[k][i] *= w[k][i];  // past the row's end g is zero
        a += g[k][i];
        b = fmaf(g[k][i], h[k][i], b);
      }
    row_sum2<kBlock>(a, b, lanes, lds[turn]);
    a *= inv;
    b *= inv;
    T* dx = static_cast<T*>(p.dx) + row * D;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; i++) g[k][i] = rstd * (g[k][i] - a - h[k][i] * b);
      store_vec<T>(dx + c, g[k], D - c);
    }
  }
  float* part = p.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int c = (k * lanes + lane) * N;
    if constexpr (kBlock) {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (c + i < D) {
          part[c + i] = dw[k][i];
          part[D + c + i] = db[k][i];
        }
    } else {
#pragma unroll
      for (int which = 0; which < 2; which++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) gather[threadIdx.x][i] = which ? db[k][i] : dw[k][i];
        __syncthreads();
        for (int t = threadIdx.x; t < lanes * N; t += kLnThreads) {
          const int col = k * lanes * N + t;
          float s = 0.0f;
          for (int r = 0; r < rows_wg; r++) s += gather[r * lanes + t / N][t % N];
          if (col < D) part[which * D + col] = s;
        }
      }
    }
  }
}

// Rows past a workgroup's registers: dw and db gather in the workgroup's own
// row of partial sums (cleared first), which stays in cache.
template <typename T, typename P>
__global__ __launch_bounds__(kLnThreads) void layer_norm_backward_long_kernel(LayerNormParams p) {
  constexpr int N = Vec16<T>::kN;
  __shared__ float lds[2][2][kLnWaves];
  const int D = p.cols;
  const float inv = 1.0f / (float)D;
  float* part = p.part + (int64_t)blockIdx.x * 2 * D;
  bool first = true;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1, first = false) {
    const T* x = static_cast<const T*>(p.x) + row * D;
    const T* dy = static_cast<const T*>(p.dy) + row * D;
    T* dx = static_cast<T*>(p.dx) + row * D;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float a = 0.0f, b = 0.0f, h[N], g[N], w[N];
    for (int c = threadIdx.x * N; c < D; c += kLnThreads * N) {
      load_vec<T>(h, x + c, D - c);
      load_vec<T>(g, dy + c, D - c);
      load_param(w, static_cast<const P*>(p.weight) + c, D - c);
#pragma unroll
      for (int i = 0; i < N; i++) {
        h[i] = (h[i] - mean) * rstd;
        if (c + i < D) {  // this thread alone owns these columns of the workgroup's row
          part[c + i] = first ? g[i] * h[i] : fmaf(g[i], h[i], part[c + i]);
          part[D + c + i] = first ? g[i] : part[D + c + i] + g[i];
        }
        g[i] *= w[i];
        a += g[i];
        b = fmaf(g[i], h[i], b);
      }
    }
    row_sum2<true>(a, b, kLnThreads, lds[turn]);
    a *= inv;
    b *= inv;
    for (int c = threadIdx.x * N; c < D; c += kLnThreads * N) {
      load_vec<T>(h, x + c, D - c);
      load_vec<T>(g, dy + c, D - c);
      load_param(w, static_cast<const P*>(p.weight) + c, D - c);
#pragma unroll
      for (int i = 0; i < N; i++) g[i] = rstd * (g[i] * w[i] - a - (h[i] - mean) * rstd * b);
      store_vec<T>(dx + c, g, D - c);
    }
  }
}

// dw and db from the partial rows: 32 columns a workgroup, 32 slices of the
// rows, joined in LDS in a fixed order.
template <typename P>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* part, int n, int D, P* dw, P* db) {
  __shared__ float lds[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float s = 0.0f;
  if (col < 2 * D) {
    int r = slice;
    for (; r + 7 * 32 < n; r += 8 * 32) {   // eight loads in flight
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = part[(int64_t)(r + i * 32) * 2 * D + col];
#pragma unroll
      for (int i = 0; i < 8; i++) s += v[i];
    }
    for (; r < n; r += 32) s += part[(int64_t)r * 2 * D + col];
  }
  lds[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && col < 2 * D) {
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; r++) t += lds[r][threadIdx.x];
    if (col < D) dw[col] = from_f32<P>(t);
    else if (db) db[col - D] = from_f32<P>(t);
  }
}

int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}

int vectors(int cols, int dtype) {
  const int n = dtype == NEST_DTYPE_F32 ? 4 : 8;
  return (cols + n - 1) / n;
}

// A row's lanes, and vectors a lane: up to 192 vectors stay with one wave (no
// barrier), up to 1024 (2048 of float32) with a workgroup of as many waves as
// they need; nv 0: past the registers.
struct LnShape {
  int lanes, nv;
  bool block;
};
//
// A forward of few rows takes a workgroup from 65 vectors on, for more loads
// in flight: 5003 x 1155 f16 13.3 us instead of 15.8 with a wave a row, while
// 50,000 rows take 73 instead of 68.
LnShape shape_of(int cols, int dtype, bool few_rows = false) {
  const int vecs = vectors(cols, dtype), most = dtype == NEST_DTYPE_F32 ? kLnMost : kLnMost / 2;
  if (vecs <= (few_rows ? 64 : 192)) return {vecs <= 64 ? pow2_at_least(vecs) : 64, (vecs + 63) / 64, false};
  if (vecs <= 2 * most) {
    const int nv = vecs <= 512 ? 1 : 2;
    return {(vecs + 64 * nv - 1) / (64 * nv) * 64, nv, true};
  }
  return {kLnThreads, 0, true};
}

// Calls f with the shape as constants.
template <typename F>
void with_shape(const LnShape& h, F f) {
  using std::integral_constant;
  if (!h.block) {
    if (h.nv == 1) f(integral_constant<int, 1>(), integral_constant<bool, false>());
    else if (h.nv == 2) f(integral_constant<int, 2>(), integral_constant<bool, false>());
    else f(integral_constant<int, 3>(), integral_constant<bool, false>());
  } else if (h.nv == 1) f(integral_constant<int, 1>(), integral_constant<bool, true>());
  else if (h.nv == 2) f(integral_constant<int, 2>(), integral_constant<bool, true>());
  else f(integral_constant<int, 0>(), integral_constant<bool, true>());
}

int64_t row_groups(int64_t rows, const LnShape& h) {
  const int rows_wg = h.block ? 1 : kLnThreads / h.lanes;
  return (rows + rows_wg - 1) / rows_wg;
}

template <typename T, typename P>
hipError_t forward(const LayerNormParams& p, hipStream_t s) {
  const LnShape h = shape_of(p.cols, p.dtype, p.rows < 16384);
  const int64_t need = row_groups(p.rows, h);
  const unsigned grid = (unsigned)(need < kLnForwardGrid ? need : kLnForwardGrid);
  with_shape(h, [&](auto nv, auto block) {
    if constexpr (nv == 0) layer_norm_long_kernel<T, P><<<grid, kLnThreads, 0, s>>>(p);
    else layer_norm_kernel<T, P, nv, block><<<grid, block ? h.lanes : kLnThreads, 0, s>>>(p, h.lanes);
  });
  return hipGetLastError();
}

template <typename T, typename P>
hipError_t backward(const LayerNormParams& p, hipStream_t s) {
  const int n = layer_norm_partials(p.rows, p.cols, p.dtype);
  if (n > 0) {
    const LnShape h = shape_of(p.cols, p.dtype);
    with_shape(h, [&](auto nv, auto block) {
      if constexpr (nv == 0) layer_norm_backward_long_kernel<T, P><<<n, kLnThreads, 0, s>>>(p);
      else layer_norm_backward_kernel<T, P, nv, block><<<n, block ? h.lanes : kLnThreads, 0, s>>>(p, h.lanes);
    });
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  layer_norm_reduce_kernel<P><<<(2 * p.cols + 31) / 32, 1024, 0, s>>>(p.part, n, p.cols, static_cast<P*>(p.dweight),
                                                                      static_cast<P*>(p.dbias));
  return hipGetLastError();
}

}  // namespace

// Workgroups of the backward: as many as the registers let run at once (waves
// a CU), so that none waits for a turn of its own.
int layer_norm_partials(int64_t rows, int cols, int dtype) {
  const LnShape h = shape_of(cols, dtype);
  const bool wide = dtype == NEST_DTYPE_F32;
  const int waves = h.block ? h.lanes / 64 : kLnThreads / 64;
  const int a_cu = h.block ? (h.nv == 1 || wide ? 16 : 8) : h.nv == 1 ? 20 : h.nv == 2 || wide ? 12 : 8;
  const int64_t need = row_groups(rows, h), most = 256 * a_cu / waves;
  return (int)(need < most ? need : most);
}

#define NEST_LN_DISPATCH(fn)                                                                                   \
  if (p.dtype == NEST_DTYPE_F32) return fn<float, float>(p, s);                                                \
  if (p.dtype == NEST_DTYPE_F16)                                                                               \
    return p.param_dtype == NEST_DTYPE_F32 ? fn<f16_t, float>(p, s) : fn<f16_t, f16_t>(p, s);                  \
  return p.param_dtype == NEST_DTYPE_F32 ? fn<bf16_t, float>(p, s) : fn<bf16_t, bf16_t>(p, s);

hipError_t launch_layer_norm(const LayerNormParams& p, hipStream_t s) { NEST_LN_DISPATCH(forward) }
hipError_t launch_layer_norm_backward(const LayerNormParams& p, hipStream_t s) { NEST_LN_DISPATCH(backward) }
#undef NEST_LN_DISPATCH

}  // namespace nest
