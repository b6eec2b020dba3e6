// The products of a gated feed-forward block as tiles of tile_gemm.h, for one
// element type.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  y = h Wd^T
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// One kernel makes g and u of the same tile (its weight tile takes 16 rows of
// Wg, then the same 16 of Wu, so both land in the same lanes), applies the
// activation and writes h; one makes dh and turns it into dg, du and h with
// the kept g and u; dx is one sum over both pairs; the three weight gradients
// share a launch.  Every product is summed in float32.  g and u are kept in
// float32, because rounding them to 16 bits would make the gradients' error
// nearly twice one rounding; h, dg and du are rounded to the inputs' type, as
// operands of the next product.
//
// Operands whose rows are no multiple of 16 bytes are copied to padded rows
// first (pad_kernel), so that the tiles have one way to load.
//
// Measured, 8192 rows, 2048 -> 8192, bf16: gate 525 us (550 GFLOP, 0.67 GB
// written), y 235, dg, du and h 385 (275 GFLOP, 0.94 GB), dx 435, the weight
// gradients 720: bound by the products (tile_gemm.h).
#pragma once

#include "blocks_internal.h"
#include "tile_gemm.h"

namespace nest {
namespace {

// ---- activations and their slopes ----

// exp and 1 / x: for 16-bit results the hardware's (1 ulp each, exp's argument
// rounded once more); for float32 the library's and a division.
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}
template <typename T>
__device__ __forceinline__ float inverse(float x) {
  if constexpr (sizeof(T) == 4) return 1.0f / x;
  return __builtin_amdgcn_rcpf(x);
}

// act(g), and its slope where it is asked for.  Phi(g) of GELU: for float32 by
// erf; for 16-bit results by Hastings' rational form (Abramowitz and Stegun
// 7.1.26, absolute error 1.5e-7 of erf), which shares exp(-g^2 / 2) with the
// slope's density.
template <typename T, int kAct, bool kSlope>
__device__ __forceinline__ float act_value(float g, float& slope) {
  if constexpr (kAct == NEST_ACT_RELU) {
    if constexpr (kSlope) slope = g > 0.0f ? 1.0f : 0.0f;
    return g <= 0.0f ? 0.0f : g;  // NaN stays
  }
  if constexpr (kAct == NEST_ACT_SILU) {
    const float q = inverse<T>(1.0f + exp_of<T>(-g));
    if constexpr (kSlope) slope = q * fmaf(g, 1.0f - q, 1.0f);
    return g * q;
  }
  float phi, e = 0.0f;
  if constexpr (sizeof(T) == 4) {
    phi = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    if constexpr (kSlope) e = expf(-0.5f * g * g);
  } else {
    const float x = fabsf(g) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
    e = exp_of<T>(-x * x);
    const float tail = 0.5f * e * t *
        fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    phi = g < 0.0f ? tail : 1.0f - tail;
  }
  if constexpr (kSlope) slope = fmaf(g * e, 0.39894228040143268f, phi);
  return g * phi;
}

// f with the activation as a constant, so that no element branches on it.
template <int kAct>
struct ActConstant {
  static constexpr int value = kAct;
};
template <typename F>
__host__ __device__ __forceinline__ auto with_act(int act, F f) {
  if (act == NEST_ACT_RELU) return f(ActConstant<NEST_ACT_RELU>());
  if (act == NEST_ACT_SILU) return f(ActConstant<NEST_ACT_SILU>());
  return f(ActConstant<NEST_ACT_GELU>());
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// Four columns n .. n + 3 of a row of N values.
template <typename T>
__device__ __forceinline__ void store4(T* row, int n, int N, bool aligned, f32x4 v) {
  if (aligned && n + 4 <= N) {
    Four<T> t;
#pragma unroll
    for (int i = 0; i < 4; i++) t.v[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Four<T>*>(row + n) = t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (n + i < N) row[n + i] = from_f32<T>(v[i]);
  }
}

// Columns n .. n + 3, those from N on as zero.
__device__ __forceinline__ f32x4 before(f32x4 v, int n, int N) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = n + e < N ? v[e] : 0.0f;
  return v;
}

// 16 x 16-column fragments of a wave to row-major rows, through LDS of its own
// so that a row's columns leave in 16-byte stores side by side.
template <typename T, int FN>
struct RowStage {
  static constexpr int kPitch = FN * 16 + 16 / (int)sizeof(T);   // elements
  T v[16 * kPitch];
};

// Rows row .. row + 15 and columns col .. col + 16 FN - 1 of out [rows][ld]; ld
// is a multiple of 16 bytes and out aligned.  Element f(j)[e] is column
// 16 j + 4 (lane / 16) + e of row lane % 16.
template <typename T, int FN, typename F>
__device__ __forceinline__ void store_rows(RowStage<T, FN>& stage, T* out, int64_t row, int64_t rows, int col, int64_t ld, F f,
                                           int lane) {
  constexpr int kVec = 16 / (int)sizeof(T), kRow = FN * 16 / kVec;
#pragma unroll
  for (int j = 0; j < FN; j++) {
    const f32x4 v = f(j);
    Four<T> t;
#pragma unroll
    for (int e = 0; e < 4; e++) t.v[e] = from_f32<T>(v[e]);
    *reinterpret_cast<Four<T>*>(&stage.v[(lane & 15) * RowStage<T, FN>::kPitch + j * 16 + (lane >> 4) * 4]) = t;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int k = lane; k < 16 * kRow; k += 64) {
    const int r = k / kRow, c = (k % kRow) * kVec;
    const uint4 v = *reinterpret_cast<const uint4*>(&stage.v[r * RowStage<T, FN>::kPitch + c]);
    if (row + r < rows && col + c < ld) *reinterpret_cast<uint4*>(out + (row + r) * ld + col + c) = v;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- C = A B (+ A2 B2), up to three products in a launch, k split over `splits` ----

template <typename T>
struct Product {
  const T *a, *b, *a2, *b2;
  int64_t lda, ldb;
  int M, N;
  int64_t K;
  T* c;               // [M][N]
  int tiles_m, tiles_n;
  int64_t part;       // offset in a slice of the partial sums
};

template <typename T>
struct Products {
  Product<T> p[3];
  int n, splits;
  float* part;        // [splits][part_size], or null where splits is 1
  int64_t part_size;
};

template <typename T, bool kAK, bool kBK, typename C>
__global__ __launch_bounds__(C::NT) void product_kernel(Products<T> all) {
  const int split = all.splits > 1 ? blockIdx.x % all.splits : 0;
  int id = all.splits > 1 ? blockIdx.x / all.splits : blockIdx.x, which = 0;
  while (which + 1 < all.n && id >= all.p[which].tiles_m * all.p[which].tiles_n) {
    id -= all.p[which].tiles_m * all.p[which].tiles_n;
    which++;
  }
  const Product<T>& p = all.p[which];
  int tm, tn;
  tile_of(id, p.tiles_m, p.tiles_n, tm, tn);
  constexpr int kStep = kStepBytes / (int)sizeof(T);
  const int64_t per = ((p.K + kStep - 1) / kStep + all.splits - 1) / all.splits * kStep;
  const int64_t k0 = split * per, k = p.K - k0 < per ? p.K - k0 : per;
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
  f32x4 acc[C::FM][C::FN] = {};
  Loader<T, kAK, C::BM, C::NT> la;
  Loader<T, kBK, C::BN, C::NT> lb;
  const int64_t ka = kAK ? k0 : k0 * p.lda, kb = kBK ? k0 : k0 * p.ldb;
  const char *a2 = nullptr, *b2 = nullptr;
  if (p.a2) {
    la.init(p.a2 + ka, p.lda, m0, kAK ? p.M : p.lda);
    lb.init(p.b2 + kb, p.ldb, n0, kBK ? p.N : p.ldb);
    a2 = la.base;
    b2 = lb.base;
  }
  la.init(p.a + ka, p.lda, m0, kAK ? p.M : p.lda);
  lb.init(p.b + kb, p.ldb, n0, kBK ? p.N : p.ldb);
  tile_product<T, kAK, kBK, C>(la, lb, k, a2, b2, acc);   // a split past the end has k <= 0: it loads zeros
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // made again here, not held in a register over the products
  const int w = wave_id();
  const int64_t m = m0 + (w / C::WN) * C::FM * 16;
  const int n = (int)n0 + (w % C::WN) * C::FN * 16;
  constexpr int kVec = 16 / (int)sizeof(T);
  if (!all.part && p.N % kVec == 0) {   // whole 16-byte pieces of the rows of C
    __syncthreads();   // the operands' LDS is free
    auto& stage = reinterpret_cast<RowStage<T, C::FN>*>(tile_lds<C>())[w];
#pragma unroll
    for (int i = 0; i < C::FM; i++)
      store_rows<T, C::FN>(stage, p.c, m + i * 16, p.M, n, p.N, [&](int j) { return acc[i][j]; }, lane);
    return;
  }
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < C::FM; i++) {
    if (m + i * 16 + r >= p.M) continue;
#pragma unroll
    for (int j = 0; j < C::FN; j++) {
      if (all.part) store4(all.part + split * all.part_size + p.part + (m + i * 16 + r) * p.N, n + j * 16 + q * 4, p.N, p.N % 4 == 0, acc[i][j]);
      else store4(p.c + (m + i * 16 + r) * p.N, n + j * 16 + q * 4, p.N, p.N % 4 == 0, acc[i][j]);
    }
  }
}

// s + the n slices of a power of two, all loads before the first sum.
template <int n>
__device__ __forceinline__ f32x4 add_slices(f32x4 s, const float* part, int64_t slice) {
  f32x4 v[n];
#pragma unroll
  for (int i = 0; i < n; i++) v[i] = *reinterpret_cast<const f32x4*>(part + i * slice);
#pragma unroll
  for (int i = 0; i < n; i++) s += v[i];
  return s;
}

// Joins the partial sums, in the order of the splits (a power of two), four
// places a thread; the products' parts of a slice are whole workgroups.
// 32 x 2048 in eight splits 3.3 us, with one load after another 4.1.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Products<T> all) {
  for (int64_t first = (int64_t)blockIdx.x * kJoinGroup; first < all.part_size; first += (int64_t)gridDim.x * kJoinGroup) {
    int which = 0;
    while (which + 1 < all.n && first >= all.p[which + 1].part) which++;
    const Product<T>& p = all.p[which];
    const int64_t e = first + threadIdx.x * 4, at = e - p.part, left = (int64_t)p.M * p.N - at;
    if (left <= 0) continue;
    const float* part = all.part + e;
    f32x4 s = {};
    if (all.splits == 2) s = add_slices<2>(s, part, all.part_size);
    else if (all.splits == 4) s = add_slices<4>(s, part, all.part_size);
    else
      for (int i = 0; i < all.splits; i += 8) s = add_slices<8>(s, part + i * all.part_size, all.part_size);
    store4(p.c + at, 0, left < 4 ? (int)left : 4, true, s);
  }
}

// ---- h = act(g) u ----

// The kept pre-activations in the order the accumulators hold them: a block of
// 16 rows and 16 columns is 1 KB of g, then 1 KB of u, lane l's four columns
// (4 (l / 16) .. + 3) of row l % 16 at 16 l.  Row-major float32 rows would be
// touched 64 bytes at a time at a stride of a whole row; on 8192 rows of 8192
// that took the backward's kernel 3.3 ms, of which 0.3 is the product.
__device__ __forceinline__ float* kept_block(float* kept, int64_t row, int col, int64_t ldh) {
  return kept + ((row >> 4) * ((ldh + 15) >> 4) + (col >> 4)) * 512 + (threadIdx.x & 63) * 4;
}

template <typename T>
struct Gate {
  const T *x, *wg, *wu;   // [M][ldx], [H][ldx]
  int64_t ldx;
  int M, H;
  int64_t ldh;            // H rounded up to 16 bytes: the pad columns are written as zeros, also in a row with an infinity
  T* h;                   // [M][ldh] or null
  float* kept;            // g and u, see kept_block; or null
  int act, tiles_m, tiles_n;
};

template <typename T, typename C>
__global__ __launch_bounds__(C::NT) void gate_kernel(Gate<T> p) {
  int tm, tn;
  tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * (C::BN / 2);
  f32x4 acc[C::FM][C::FN] = {};
  Loader<T, true, C::BM, C::NT> la;
  Loader<T, true, C::BN, C::NT> lb;
  la.init(p.x, p.ldx, m0, p.M);
  lb.init_pair(p.wg, p.wu, p.ldx, n0, p.H);
  tile_product<T, true, true, C>(la, lb, p.ldx, nullptr, nullptr, acc);
  const int w = wave_id();
  const int64_t m = m0 + (w / C::WN) * C::FM * 16;
  const int n = (int)n0 + (w % C::WN) * C::FN * 8;
  if (p.kept) {
#pragma unroll
    for (int i = 0; i < C::FM; i++)
#pragma unroll
      for (int j = 0; j < C::FN; j += 2) {
        if (m + i * 16 >= p.M || n + j * 8 >= p.ldh) continue;
        float* at = kept_block(p.kept, m + i * 16, n + j * 8, p.ldh);
        *reinterpret_cast<f32x4*>(at) = acc[i][j];
        *reinterpret_cast<f32x4*>(at + 256) = acc[i][j + 1];
      }
  }
  if (!p.h) return;
  const int lane = threadIdx.x & 63;
  __syncthreads();   // the operands' LDS is free
  auto& stage = reinterpret_cast<RowStage<T, C::FN / 2>*>(tile_lds<C>())[w];
  with_act(p.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < C::FM; i++)
      store_rows<T, C::FN / 2>(stage, p.h, m + i * 16, p.M, n, p.ldh, [&](int j) {
        f32x4 h;
        float unused;
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = act_value<T, act.value, false>(acc[i][2 * j][e], unused) * acc[i][2 * j + 1][e];
        return n + j * 16 + 16 > p.H ? before(h, n + j * 16 + (lane >> 4) * 4, p.H) : h;
      }, lane);
  });
}

// ---- dg, du and h from dh = dy Wd ----

template <typename T>
struct GateBackward {
  const T *dy, *wd;       // [M][ldy], [O][ldh]
  int64_t ldy, ldh;
  int M, O, H;
  float* kept;
  T *h, *dg, *du;         // [M][ldh]; the pad columns of dg and du are zeros
  int act, tiles_m, tiles_n;
};

template <typename T, typename C>
__global__ __launch_bounds__(C::NT) void gate_backward_kernel(GateBackward<T> p) {
  int tm, tn;
  tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
  f32x4 acc[C::FM][C::FN] = {};
  Loader<T, true, C::BM, C::NT> la;
  Loader<T, false, C::BN, C::NT> lb;
  la.init(p.dy, p.ldy, m0, p.M);
  lb.init(p.wd, p.ldh, n0, p.ldh);
  tile_product<T, true, false, C>(la, lb, p.O, nullptr, nullptr, acc);
  const int w = wave_id();
  const int64_t m = m0 + (w / C::WN) * C::FM * 16;
  const int n = (int)n0 + (w % C::WN) * C::FN * 16;
  __syncthreads();   // the operands' LDS is free
  auto& stage = reinterpret_cast<RowStage<T, C::FN>*>(tile_lds<C>())[w];
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // made again here, not held in a register over the products
  with_act(p.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < C::FM; i++) {
      const int64_t row = m + i * 16;
      if (row >= p.M) break;
      f32x4 g[C::FN], u[C::FN];
#pragma unroll
      for (int j = 0; j < C::FN; j++) {
        g[j] = u[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (n + j * 16 >= p.ldh) continue;
        const float* at = kept_block(p.kept, row, n + j * 16, p.ldh);
        g[j] = *reinterpret_cast<const f32x4*>(at);
        u[j] = *reinterpret_cast<const f32x4*>(at + 256);
      }
#pragma unroll
      for (int j = 0; j < C::FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {   // g: h, u: dg, acc: du
          float slope;
          const float a = act_value<T, act.value, true>(g[j][e], slope), d = acc[i][j][e], h = a * u[j][e];
          u[j][e] = d * u[j][e] * slope;
          acc[i][j][e] = d * a;
          g[j][e] = h;
        }
      if (n + C::FN * 16 > p.H) {
#pragma unroll
        for (int j = 0; j < C::FN; j++) {
          u[j] = before(u[j], n + j * 16 + (lane >> 4) * 4, p.H);
          acc[i][j] = before(acc[i][j], n + j * 16 + (lane >> 4) * 4, p.H);
        }
      }
      store_rows<T, C::FN>(stage, p.h, row, p.M, n, p.ldh, [&](int j) { return g[j]; }, lane);
      store_rows<T, C::FN>(stage, p.dg, row, p.M, n, p.ldh, [&](int j) { return u[j]; }, lane);
      store_rows<T, C::FN>(stage, p.du, row, p.M, n, p.ldh, [&](int j) { return acc[i][j]; }, lane);
    }
  });
}

// ---- padded copies ----

template <typename T>
struct Pads {
  const T* from[5];
  T* to[5];
  int64_t rows[5];
  int n[5], ld[5];   // row lengths
};

template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(Pads<T> p) {
  constexpr int N = Vec16<T>::kN;
  const int k = blockIdx.y, n = p.n[k], chunks = p.ld[k] / N;
  const int64_t total = p.rows[k] * chunks;
  const bool small = total < (int64_t)1 << 32;   // a division of 32 bits does
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = small ? (int64_t)((uint32_t)i / (uint32_t)chunks) : i / chunks;
    const int c = (int)(i - row * chunks) * N;
    float v[N];
    load_vec<T>(v, p.from[k] + row * n + c, n - c);
    store_vec<T>(p.to[k] + row * p.ld[k] + c, v, N);
  }
}

// ---- the choice of tiles, and launches ----

// f with the tile of a launch of `groups` workgroups.
template <typename F>
void with_tile(int side, int64_t groups, F f) {
  if (side == 256) f(TileL());
  else if (side == 128) f(TileM());
  else groups <= kMoreBuffers ? f(TileS4()) : f(TileS());
}

template <typename T, bool kAK, bool kBK>
hipError_t launch_products(Products<T>& all, TileChoice t, hipStream_t s) {
  int64_t tiles = 0, part = 0;
  for (int i = 0; i < all.n; i++) {
    all.p[i].tiles_m = (int)tiles_along(all.p[i].M, t.side);
    all.p[i].tiles_n = (int)tiles_along(all.p[i].N, t.side);
    all.p[i].part = part;
    tiles += (int64_t)all.p[i].tiles_m * all.p[i].tiles_n;
    part += ((int64_t)all.p[i].M * all.p[i].N + kJoinGroup - 1) / kJoinGroup * kJoinGroup;
  }
  all.splits = t.splits;
  all.part_size = part;
  if (t.splits == 1) all.part = nullptr;
  const unsigned grid = (unsigned)(tiles * t.splits);
  with_tile(t.side, grid, [&](auto c) {
    typedef decltype(c) C;
    static_assert(C::NT == tile_threads(C::BM), "");
    product_kernel<T, kAK, kBK, C><<<grid, C::NT, 0, s>>>(all);
  });
  if (t.splits > 1) {
    const int64_t need = part / kJoinGroup;
    join_kernel<T><<<(unsigned)(need < 65536 ? need : 65536), 256, 0, s>>>(all);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_gate(Gate<T> p, TileChoice t, hipStream_t s) {
  p.tiles_m = (int)tiles_along(p.M, t.side);
  p.tiles_n = (int)tiles_along(p.ldh, t.side / 2);
  const unsigned grid = (unsigned)((int64_t)p.tiles_m * p.tiles_n);
  with_tile(t.side, grid, [&](auto c) {
    typedef decltype(c) C;
    gate_kernel<T, C><<<grid, C::NT, 0, s>>>(p);
  });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_gate_backward(GateBackward<T> p, TileChoice t, hipStream_t s) {
  p.tiles_m = (int)tiles_along(p.M, t.side);
  p.tiles_n = (int)tiles_along(p.ldh, t.side);
  const unsigned grid = (unsigned)((int64_t)p.tiles_m * p.tiles_n);
  with_tile(t.side, grid, [&](auto c) {
    typedef decltype(c) C;
    gate_backward_kernel<T, C><<<grid, C::NT, 0, s>>>(p);
  });
  return hipGetLastError();
}

// The padded operands of a call: x and the weights, dy in a backward.
template <typename T>
struct Operands {
  const T *x, *wg, *wu, *wd, *dy;
};

template <typename T>
hipError_t pad_operands(const GatedParams& p, const GatedLayout& l, uint8_t* ws, bool back, Operands<T>& o, hipStream_t s) {
  o = {static_cast<const T*>(p.x), static_cast<const T*>(p.w_gate), static_cast<const T*>(p.w_up),
       static_cast<const T*>(p.w_down), static_cast<const T*>(p.dy)};
  Pads<T> q{};
  int n = 0;
  int64_t most = 0;
  auto add = [&](const T*& src, size_t at, int64_t rows, int len, int64_t ld) {
    T* to = reinterpret_cast<T*>(ws + at);
    q.from[n] = src;
    q.to[n] = to;
    q.rows[n] = rows;
    q.n[n] = len;
    q.ld[n++] = (int)ld;
    if (rows * ld > most) most = rows * ld;
    src = to;
  };
  if (l.ldx != p.in) {
    add(o.x, l.x, p.rows, p.in, l.ldx);
    add(o.wg, l.wg, p.hidden, p.in, l.ldx);
    add(o.wu, l.wu, p.hidden, p.in, l.ldx);
  }
  if (l.ldh != p.hidden) add(o.wd, l.wd, p.out, p.hidden, l.ldh);
  if (back && l.ldy != p.out) add(o.dy, l.dy, p.rows, p.out, l.ldy);
  if (n) {
    const int64_t need = (most / Vec16<T>::kN + 255) / 256;
    pad_kernel<T><<<dim3((unsigned)(need < 4096 ? need : 4096), n), 256, 0, s>>>(q);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace nest
