// A branch joined to the residual stream between two root-mean-square norms,
// and its backward pass.
//
//   a = 1 / sqrt(sum h^2 / D + eps),  t^ = a h,  t = t^ post
//   r = scale x + gate t              (rounded: the stream as it is stored)
//   c = 1 / sqrt(sum r^2 / D + eps),  r^ = c r,  y = r^ pre
//
//   p = dy pre,  e = dr + c (p - r^ sum(p r^) / D),  dx = scale e
//   q = e gate post,  dh = a (q - t^ sum(q t^) / D)
//   dgate = sum e t,  dpost = sum e gate t^,  dpre = sum dy r^
//
// Memory bound: forward reads x and h and writes r and y, backward reads dr,
// dy, r and h and writes dx and dh, each once.  A row is held in registers
// over both of its sums.  y is the norm of r as it is stored, in the streams'
// type: what follows reads that r too, and the backward pass makes the same r^
// from it.  All sums are float32; every result is rounded once.  1,702,400 x 64
// of bf16: forward 166 us (872 MB: 5.3 TB/s), backward 273 (1308 MB: 4.8 TB/s);
// 8192 x 4096 of float32 with 8 gates 101 (5.3 TB/s) and 175 (4.6 TB/s).
//
// A row of up to 64 vectors of 16 bytes (backward 128) belongs to 1 to 64 lanes
// of a wave, a longer one to a workgroup.  A gate is shared by consecutive rows; in the
// backward pass an item is a part of the rows of one gate, and what its lanes
// gather, S = sum e t^, gives both dgate = post S and its share gate S of
// dpost, which gathers on over the items of a workgroup where there are several
// gates.  Where every row has a gate of its own, dgate is written row by row
// and dpost is gathered.  Sums over rows are joined in an order that the
// sizes fix.
#include "column_sums.h"
#include "residual_internal.h"

#include <type_traits>

namespace nest {
namespace {

constexpr int kThreads = 256;        // of rows that stay with a wave
constexpr int kMostThreads = 512;    // that share a row: 16 values a lane at most
constexpr int kMostWaves = kMostThreads / 64;
constexpr int64_t kForwardGrid = 2048;   // workgroups

// Sums over the lanes of a row; every lane gets the result.  Two LDS buffers
// in turn: one barrier a sum is enough.
template <bool kBlock>
struct RowSum {
  float (*lds)[kMostWaves];
  int turn = 0;
  __device__ __forceinline__ float operator()(float v, int lanes) {
    if constexpr (kBlock) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
      if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = v;
      __syncthreads();
      v = 0.0f;
      for (int w = 0; w < (int)blockDim.x / 64; w++) v += lds[turn][w];
      turn ^= 1;
    } else {
      for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    }
    return v;
  }
};

// N parameters as they lie in memory: a load whose wait comes at its use.
template <typename P, int N>
struct ParamVec {
  static constexpr int K = Vec16<P>::kN;
  static_assert(N % K == 0, "");
  Words16<P> v[N / K];
  __device__ __forceinline__ void load(const P* p, int n) {
#pragma unroll
    for (int k = 0; k < N / K; k++) v[k] = load_words<false>(p + k * K, n - k * K);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32(v[i / K][i % K]); }
};

// Parameters of this lane's columns, `other` where there are none.
template <typename P, int NV, int N>
__device__ __forceinline__ void load_columns(float (&w)[NV][N], const void* p, int lane, int lanes, int D, float other) {
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int c = (k * lanes + lane) * N;
    if (p) {
      load_param(w[k], static_cast<const P*>(p) + c, D - c);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) w[k][i] = other;
    }
  }
}

template <typename T, typename P, int NV, bool kBlock>
__global__ __launch_bounds__((kBlock ? kMostThreads : kThreads)) void residual_norm_kernel(ResidualNormParams p, int lanes,
                                                                                            uint32_t rows_gate) {
  constexpr int N = Vec16<T>::kN;
  __shared__ float lds[2][kMostWaves];
  RowSum<kBlock> sum{lds};
  const int rows_wg = kBlock ? 1 : kThreads / lanes;
  const int lane = kBlock ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int D = p.cols;
  const float inv = 1.0f / (float)D;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  int64_t row = (int64_t)blockIdx.x * rows_wg + (kBlock ? 0 : threadIdx.x / lanes);
  const bool row_gates = p.gate && p.gates > 1;
  Words16<T> nx[NV], nh[NV];
  ParamVec<P, N> ng[NV];
  auto load = [&](int64_t at) {
    const bool in = at < p.rows;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N, n = in ? D - c : 0;
      nx[k] = load_words<false>(static_cast<const T*>(p.x) + at * D + c, n);
      if (p.h) nh[k] = load_words<false>(static_cast<const T*>(p.h) + at * D + c, n);
      if (row_gates) ng[k].load(static_cast<const P*>(p.gate) + (int64_t)((uint32_t)at / rows_gate) * D + c, n);
    }
  };
  load(row);
  float post[NV][N], pre[NV][N], gate[NV][N];
  load_columns<P>(post, p.post, lane, lanes, D, 1.0f);
  load_columns<P>(pre, p.pre, lane, lanes, D, 0.0f);
  load_columns<P>(gate, row_gates ? nullptr : p.gate, lane, lanes, D, 1.0f);
  for (; row < p.rows; row += step) {   // in kBlock the same number of turns for all threads
    float r[NV][N], t[NV][N];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        r[k][i] = to_f32(nx[k][i]);
        if (p.h) {
          t[k][i] = to_f32(nh[k][i]);
          s = fmaf(t[k][i], t[k][i], s);
          if (row_gates) gate[k][i] = ng[k][i];
        }
      }
    load(row + step);   // on its way while this row is worked on
    if (p.h) {
      float a = 1.0f;
      if (p.post) {
        a = 1.0f / sqrtf(sum(s, lanes) * inv + p.eps);
        if (lane == 0 && p.rstd_post) p.rstd_post[row] = a;
      }
      s = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * lanes + lane) * N;
        Vec16<T> out;
#pragma unroll
        for (int i = 0; i < N; i++) {
          out.v[i] = from_f32<T>(fmaf(t[k][i] * a * post[k][i], gate[k][i], p.scale * r[k][i]));
          r[k][i] = to_f32(out.v[i]);
        }
        store_raw(static_cast<T*>(p.r) + row * D + c, out, D - c);
      }
    }
    if (!p.pre) continue;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) s = fmaf(r[k][i], r[k][i], s);
    const float c0 = 1.0f / sqrtf(sum(s, lanes) * inv + p.eps);
    if (lane == 0 && p.rstd_pre) p.rstd_pre[row] = c0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = (k * lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; i++) r[k][i] = r[k][i] * c0 * pre[k][i];
      store_vec<T>(static_cast<T*>(p.y) + row * D + c, r[k], D - c);
    }
  }
}

// What a lane gathered for its columns, as a row of float32 sums; the rows of
// a workgroup that share columns are added in their order.
template <int NV, int N, bool kBlock>
__device__ __forceinline__ void write_sums(const float (&v)[NV][N], float* out, int lane, int lanes, int D, float (*gather)[N + 1]) {
#pragma unroll
  for (int k = 0; k < NV; k++) {
    if constexpr (kBlock) {
      const int c = (k * lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; i++)
        if (c + i < D) out[c + i] = v[k][i];
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; i++) gather[threadIdx.x][i] = v[k][i];
      __syncthreads();
      for (int t = threadIdx.x; t < lanes * N; t += kThreads) {
        const int col = k * lanes * N + t;
        float s = 0.0f;
        for (int r = 0; r < kThreads / lanes; r++) s += gather[r * lanes + t / N][t % N];
        if (col < D) out[col] = s;
      }
    }
  }
}

// Items: `parts` parts of the rows of each gate (one gate for all rows where
// there is none, or one a row: kEachRow).  A workgroup takes every
// gridDim.x-th; it writes a row of S an item, one row of dpre and, with
// several gates (kSeveral), one of dpost.
struct Items {
  int64_t rows;       // of a gate
  int64_t n;          // items
  int parts;          // of a gate
  float *s, *dpre, *dpost;
};
enum Gates { kOneGate, kSeveral, kEachRow };
// Waves a SIMD that the registers leave room for: four where asked to.
constexpr bool four_waves(int nv, int values, bool block, Gates gates) { return nv * values <= 8 && (nv == 1 || block) && gates != kEachRow; }

template <typename T, typename P, int NV, bool kBlock, Gates kGates>
__global__ __launch_bounds__((kBlock ? kMostThreads : kThreads), (four_waves(NV, Vec16<T>::kN, kBlock, kGates) ? 4 : 1)) void
residual_norm_backward_kernel(ResidualNormParams p, int lanes, Items items) {
  constexpr int N = Vec16<T>::kN;
  constexpr bool kEach = kGates == kEachRow;
  constexpr bool kAhead = NV * N < 16;   // a row's gate loaded with the row before; past the registers else
  __shared__ float lds[2][kMostWaves];
  __shared__ float gather[kBlock ? 1 : kThreads][N + 1];
  RowSum<kBlock> sum{lds};
  const int rows_wg = kBlock ? 1 : kThreads / lanes;
  const int lane = kBlock ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int D = p.cols;
  const float inv = 1.0f / (float)D;
  float w[NV][N], pre[NV][N], gate[NV][N], acc[NV][N], dpre[NV][N];   // w: post, times the item's gate unless every row has its own
  __shared__ float dpost[kGates == kSeveral ? NV * N : 1][kBlock ? kMostThreads : kThreads];   // each thread's own: registers would cost a wave a SIMD
  if constexpr (kGates == kSeveral) {
#pragma unroll
    for (int i = 0; i < NV * N; i++) dpost[i][threadIdx.x] = 0.0f;
  }
  if constexpr (kEach) load_columns<P>(w, p.post, lane, lanes, D, 1.0f);
  load_columns<P>(pre, p.pre, lane, lanes, D, 0.0f);
#pragma unroll
  for (int k = 0; k < NV; k++)
#pragma unroll
    for (int i = 0; i < N; i++) dpre[k][i] = 0.0f;
  for (int64_t item = blockIdx.x; item < items.n; item += gridDim.x) {
    const int64_t group = item / items.parts;
    const int64_t first = group * items.rows, last = first + items.rows;
    const int64_t step = (int64_t)items.parts * rows_wg;
    int64_t row = first + (item - group * items.parts) * rows_wg + (kBlock ? 0 : threadIdx.x / lanes);
    if constexpr (!kEach) {
      load_columns<P>(w, p.post, lane, lanes, D, 1.0f);
      load_columns<P>(gate, p.gate ? static_cast<const P*>(p.gate) + group * D : nullptr, lane, lanes, D, 1.0f);
    }
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        if constexpr (!kEach) w[k][i] *= gate[k][i];
        acc[k][i] = 0.0f;
      }
    Words16<T> nr[NV], nh[NV], ndr[NV], ndy[NV];
    ParamVec<P, N> ng[NV];
    float na = 1.0f, nc = 0.0f;
    auto load = [&](int64_t at) {
      const bool in = at < last;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * lanes + lane) * N, n = in ? D - c : 0;
        if (p.pre) nr[k] = load_words<false>(static_cast<const T*>(p.r) + at * D + c, n);
        if (p.h) nh[k] = load_words<false>(static_cast<const T*>(p.h) + at * D + c, n);
        ndr[k] = load_words<false>(static_cast<const T*>(p.dr) + at * D + c, p.dr ? n : 0);
        if (p.pre) ndy[k] = load_words<false>(static_cast<const T*>(p.dy) + at * D + c, p.dy ? n : 0);
        if constexpr (kEach && kAhead) ng[k].load(static_cast<const P*>(p.gate) + at * D + c, n);
      }
      if (in && p.post) na = p.rstd_post[at];
      if (in && p.pre) nc = p.rstd_pre[at];
    };
    load(row);
    for (; row < last; row += step) {
      float e[NV][N], hat[NV][N];
      const float a = na, c0 = nc;
      float s = 0.0f;
      if (p.pre) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int i = 0; i < N; i++) {
            const float g = to_f32(ndy[k][i]);
            hat[k][i] = to_f32(nr[k][i]) * c0;
            dpre[k][i] = fmaf(g, hat[k][i], dpre[k][i]);
            e[k][i] = g * pre[k][i];   // past the row's end zero
            s = fmaf(e[k][i], hat[k][i], s);
          }
        s = sum(s, lanes) * inv;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int i = 0; i < N; i++) e[k][i] = fmaf(c0, e[k][i] - hat[k][i] * s, to_f32(ndr[k][i]));
      } else {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int i = 0; i < N; i++) e[k][i] = to_f32(ndr[k][i]);
      }
      if (p.h) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int i = 0; i < N; i++) {
            hat[k][i] = to_f32(nh[k][i]) * a;
            if constexpr (kEach && kAhead) gate[k][i] = ng[k][i];
          }
      }
      if constexpr (kEach && !kAhead) load_columns<P>(gate, static_cast<const P*>(p.gate) + row * D, lane, lanes, D, 0.0f);
      load(row + step);   // on its way while this row is worked on
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * lanes + lane) * N;
        float dx[N];
#pragma unroll
        for (int i = 0; i < N; i++) dx[i] = p.scale * e[k][i];
        store_vec<T>(static_cast<T*>(p.dx) + row * D + c, dx, D - c);
      }
      if (!p.h) continue;
      s = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * lanes + lane) * N;
        if constexpr (kEach) {
          float dg[N];
#pragma unroll
          for (int i = 0; i < N; i++) dg[i] = e[k][i] * (hat[k][i] * w[k][i]);
          store_param<P>(static_cast<P*>(p.dgate) + row * D + c, dg, D - c);
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
          if constexpr (kEach) e[k][i] *= gate[k][i];
          acc[k][i] = fmaf(e[k][i], hat[k][i], acc[k][i]);
          e[k][i] *= w[k][i];
          s = fmaf(e[k][i], hat[k][i], s);
        }
      }
      if (p.post) {
        s = sum(s, lanes) * inv;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int i = 0; i < N; i++) e[k][i] = a * (e[k][i] - hat[k][i] * s);
      }
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int c = (k * lanes + lane) * N;
        store_vec<T>(static_cast<T*>(p.dh) + row * D + c, e[k], D - c);
      }
    }
    if (items.s) write_sums<NV, N, kBlock>(acc, items.s + item * D, lane, lanes, D, gather);
    if constexpr (kGates == kSeveral) {
      load_columns<P>(gate, static_cast<const P*>(p.gate) + group * D, lane, lanes, D, 1.0f);   // again: not held over the rows
#pragma unroll
      for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < N; i++) dpost[k * N + i][threadIdx.x] += gate[k][i] * acc[k][i];
    }
  }
  if constexpr (kGates == kSeveral) {
    if (items.dpost) {
#pragma unroll
      for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < N; i++) acc[k][i] = dpost[k * N + i][threadIdx.x];
      write_sums<NV, N, kBlock>(acc, items.dpost + (int64_t)blockIdx.x * D, lane, lanes, D, gather);
    }
  }
  if (p.pre) write_sums<NV, N, kBlock>(dpre, items.dpre + (int64_t)blockIdx.x * D, lane, lanes, D, gather);
}

int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}

// A row's lanes, and vectors a lane.  Up to 64 vectors stay with one wave, in
// the backward pass up to 128 (no barrier), more with a workgroup of as many
// waves as they need.  us of 65,536 x 768 bf16 with a wave and with a workgroup
// a row: forward 120 and 106, backward 123 and 179; 16,384 x 1024 33 and 28, 40
// and 45.
struct Shape {
  int lanes, nv;
  bool block;
};
Shape shape_of(int cols, int dtype, bool back) {
  const int n = dtype == NEST_DTYPE_F32 ? 4 : 8, vecs = (cols + n - 1) / n;
  if (vecs <= (back ? 128 : 64)) return {vecs <= 64 ? pow2_at_least(vecs) : 64, (vecs + 63) / 64, false};
  const int nv = vecs <= kMostThreads ? 1 : vecs <= 2 * kMostThreads ? 2 : 4;   // 4: float32 alone
  return {(vecs + 64 * nv - 1) / (64 * nv) * 64, nv, true};
}

template <typename T, bool kBack, typename F>
void with_shape(const Shape& h, F f) {
  using std::integral_constant;
  if (!h.block) {
    if (!kBack || h.nv == 1) f(integral_constant<int, 1>(), integral_constant<bool, false>());
    else if constexpr (kBack) f(integral_constant<int, 2>(), integral_constant<bool, false>());
  } else if (h.nv == 1) f(integral_constant<int, 1>(), integral_constant<bool, true>());
  else if (sizeof(T) == 2 || h.nv == 2) f(integral_constant<int, 2>(), integral_constant<bool, true>());
  else if constexpr (sizeof(T) == 4) f(integral_constant<int, 4>(), integral_constant<bool, true>());
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int rows_of_group(const Shape& h) { return h.block ? 1 : kThreads / h.lanes; }

// The backward's items and workgroups: as many as run at once, so that none
// waits for a turn of its own and few partial sums are left to join.
struct Plan {
  Items items;
  int groups;                       // workgroups
  Gates gates;
  size_t s, dpre, dpost, floats;    // into the workspace
};
Plan plan_of(int64_t rows, int cols, int dtype, int64_t gates) {
  Plan l{};
  l.gates = gates <= 1 ? kOneGate : gates == rows ? kEachRow : kSeveral;
  const Shape h = shape_of(cols, dtype, true);
  const int waves = h.block ? h.lanes / 64 : kThreads / 64, n = dtype == NEST_DTYPE_F32 ? 4 : 8;
  const int values = h.nv * n;   // a lane's
  const int a_cu = values == 4 ? 20 : values == 8 ? (four_waves(h.nv, n, h.block, l.gates) ? 16 : 12) : 8;   // waves, by the registers
  const int64_t most = 256 * (a_cu > waves ? a_cu / waves : 1);
  const int64_t shared = l.gates == kSeveral ? gates : 1;
  l.items.rows = rows / shared;
  const int64_t turns = cdiv(l.items.rows, rows_of_group(h)), share = most / shared > 1 ? most / shared : 1;
  l.items.parts = (int)(turns < share ? turns : share);
  l.items.n = shared * l.items.parts;
  l.groups = (int)(l.items.n < most ? l.items.n : most);
  l.s = 0;
  l.dpre = (size_t)l.items.n * cols;
  l.dpost = l.dpre + (size_t)l.groups * cols;
  l.floats = l.dpost + (l.gates == kSeveral ? (size_t)l.groups * cols : 0);
  return l;
}

template <typename T, typename P>
hipError_t forward(const ResidualNormParams& p, hipStream_t s) {
  const Shape h = shape_of(p.cols, p.dtype, false);
  const int64_t need = cdiv(p.rows, rows_of_group(h));
  const unsigned grid = (unsigned)(need < kForwardGrid ? need : kForwardGrid);
  const uint32_t rows_gate = p.gates > 1 ? (uint32_t)(p.rows / p.gates) : 1;
  with_shape<T, false>(h, [&](auto nv, auto block) {
    residual_norm_kernel<T, P, nv, block><<<grid, block ? h.lanes : kThreads, 0, s>>>(p, h.lanes, rows_gate);
  });
  return hipGetLastError();
}

template <typename T, typename P>
hipError_t backward(const ResidualNormParams& p, hipStream_t s) {
  Plan l = plan_of(p.rows, p.cols, p.dtype, p.gates);
  const bool gate = p.h && p.gate, post = p.h && p.post;
  l.items.s = post || (gate && l.gates != kEachRow) ? p.ws + l.s : nullptr;
  l.items.dpre = p.ws + l.dpre;
  l.items.dpost = post && l.gates == kSeveral ? p.ws + l.dpost : nullptr;
  if (l.groups > 0) {
    const Shape h = shape_of(p.cols, p.dtype, true);
    with_shape<T, true>(h, [&](auto nv, auto block) {
      const int threads = block ? h.lanes : kThreads;
      if (l.gates == kEachRow) residual_norm_backward_kernel<T, P, nv, block, kEachRow><<<l.groups, threads, 0, s>>>(p, h.lanes, l.items);
      else if (l.gates == kSeveral) residual_norm_backward_kernel<T, P, nv, block, kSeveral><<<l.groups, threads, 0, s>>>(p, h.lanes, l.items);
      else residual_norm_backward_kernel<T, P, nv, block, kOneGate><<<l.groups, threads, 0, s>>>(p, h.lanes, l.items);
    });
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  SumTasks tasks{};
  int n = 0;
  if (p.pre) tasks.t[n++] = {l.items.dpre, l.groups, 1, p.cols, nullptr, nullptr, p.dpre, nullptr};
  if (l.items.s && l.gates == kEachRow) {
    tasks.t[n++] = {l.items.s, l.items.n, 1, p.cols, nullptr, nullptr, p.dpost, nullptr};
  } else if (l.items.s && l.gates == kSeveral) {
    tasks.t[n++] = {l.items.s, l.items.parts, p.gates, p.cols, p.post, nullptr, p.dgate, nullptr};
    if (post) tasks.t[n++] = {l.items.dpost, l.groups, 1, p.cols, nullptr, nullptr, p.dpost, nullptr};
  } else if (l.items.s) {
    tasks.t[n++] = {l.items.s, l.items.n, 1, p.cols, p.post, p.gate, gate ? p.dgate : nullptr, post ? p.dpost : nullptr};
  }
  return n ? launch_column_sums<P>(tasks, n, s) : hipSuccess;
}

}  // namespace

size_t residual_norm_ws_bytes(int64_t rows, int cols, int dtype, int64_t gates) {
  return plan_of(rows, cols, dtype, gates).floats * sizeof(float);
}

#define NEST_RN_DISPATCH(fn)                                                                                   \
  if (p.dtype == NEST_DTYPE_F32) return fn<float, float>(p, s);                                                \
  if (p.dtype == NEST_DTYPE_F16)                                                                               \
    return p.param_dtype == NEST_DTYPE_F32 ? fn<f16_t, float>(p, s) : fn<f16_t, f16_t>(p, s);                  \
  return p.param_dtype == NEST_DTYPE_F32 ? fn<bf16_t, float>(p, s) : fn<bf16_t, bf16_t>(p, s);

hipError_t launch_residual_norm(const ResidualNormParams& p, hipStream_t s) { NEST_RN_DISPATCH(forward) }
hipError_t launch_residual_norm_backward(const ResidualNormParams& p, hipStream_t s) { NEST_RN_DISPATCH(backward) }
#undef NEST_RN_DISPATCH

}  // namespace nest
