// The gated feed-forward block for narrow rows (at most 128 features in and
// out) of a 16-bit type: whole rows stay in registers from x to y.
//
// A frame has a million rows of 16 to 128 features, so the weights fit LDS and
// the block is bound by reading x and writing y once all between stays on the
// chip: h [rows][hidden] through HBM would be two to four times that traffic.
// A wave takes 16 RG rows.  It computes transposed products, weights as the
// first operand and rows as the second: the accumulators of g and u then hold
// four consecutive hidden features of one row a lane, which after the
// activation is the second operand of the next product (32 hidden features in
// the order 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3 for the lanes of
// quarter q; the down projection's weights lie in LDS in that order).
//
// Measured, 1,702,400 x 64, hidden 128: 122 us with SiLU (3.6 TB/s of x and y),
// 98 us with ReLU (4.4); the vector ALU is busy 0.74 of the time (an exponential
// and a reciprocal, 16 cycles each, for every hidden feature), the matrix cores
// 0.35.
#pragma once

#include "gated_tiles.h"

namespace nest {
namespace {

template <typename T>
struct Narrow {
  const T *x, *wg, *wu, *wd;
  T* y;
  int64_t rows;
  int in, hidden, out, act;
};

template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag load8(const T* p, int n) {
  typename Mma<T>::Frag f;
  if (n >= 8) {
    __builtin_memcpy(&f, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = i < n ? p[i] : (T)0.0f;
  }
  return f;
}

// kEnds: the hidden features end inside the last 32; h past the last one is
// zero, where an infinity times its weights of zero would make the row NaN.
template <typename T, int kAct, int KI, int RG, bool kEnds>
__global__ __launch_bounds__(512, KI <= 2 ? 4 : 2) void narrow_forward_kernel(Narrow<T> p, int chunk) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int FO = 2 * KI;
  extern __shared__ __attribute__((aligned(16))) uint8_t narrow_mem[];
  T* lds = reinterpret_cast<T*>(narrow_mem);
  const int waves = blockDim.x >> 6;
  const NarrowLds l = narrow_lds(KI, chunk, waves);
  const int h32 = (p.hidden + 31) & ~31;
  // weights of hidden features from h0 on; what lies past a matrix is zero
  auto load_weights = [&](int h0) {
    for (int c = threadIdx.x; c < 2 * chunk * (KI * 4); c += blockDim.x) {
      const int row = c / (KI * 4), k = c % (KI * 4) * 8;
      const int h = h0 + (row >> 6) * 32 + (row & 31);
      const T* w = row & 32 ? p.wu : p.wg;
      *reinterpret_cast<Frag*>(lds + row * l.pitch_in + k) = load8<T>(w + (int64_t)h * p.in + k, h < p.hidden ? p.in - k : 0);
    }
    for (int c = threadIdx.x; c < KI * 32 * (chunk / 8); c += blockDim.x) {
      const int o = c / (chunk / 8), k = c % (chunk / 8) * 8;   // elements k .. k + 7 of a row in LDS: a quarter's
      const int base = h0 + (k & ~31) + ((k >> 3) & 3) * 4;
      Frag f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int h = base + (e & 3) + (e >> 2) * 16;
        f[e] = o < p.out && h < p.hidden ? p.wd[(int64_t)o * p.hidden + h] : (T)0.0f;
      }
      *reinterpret_cast<Frag*>(lds + l.down + o * l.pitch_h + k) = f;
    }
    __syncthreads();
  };
  const bool whole = chunk >= h32;
  if (whole) load_weights(0);
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const T* w_in = lds + r * l.pitch_in + q * 8;
  const T* w_down = lds + l.down + r * l.pitch_h + q * 8;
  auto& stage = *reinterpret_cast<RowStage<T, FO>*>(lds + l.stage + wave_id() * 16 * RowStage<T, FO>::kPitch);
  // every wave of a workgroup takes the same number of turns: there may be barriers inside
  const int64_t step = (int64_t)gridDim.x * waves * (16 * RG);
  int64_t base = (int64_t)blockIdx.x * waves * (16 * RG);
  int64_t row = base + wave_id() * (16 * RG);
  Frag x[RG][KI];
  auto load_x = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < RG; i++)
#pragma unroll
      for (int k = 0; k < KI; k++) {
        const int64_t n = at + i * 16 + r;
        x[i][k] = load8<T>(p.x + n * p.in + k * 32 + q * 8, n < p.rows ? p.in - k * 32 - q * 8 : 0);
      }
  };
  load_x(row);
  for (; base < p.rows; base += step, row += step) {
    f32x4 y[RG][FO] = {};
    for (int h0 = 0; h0 < h32; h0 += chunk) {
      if (!whole) {
        __syncthreads();   // the last chunk is no longer read
        load_weights(h0);
      }
      const int end = h32 - h0 < chunk ? h32 - h0 : chunk;
      for (int hc = 0; hc < end; hc += 32) {
        f32x4 g[RG][2] = {}, u[RG][2] = {};
        const T* w = w_in + hc * 2 * l.pitch_in;
#pragma unroll
        for (int k = 0; k < KI; k++)
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const Frag fg = *reinterpret_cast<const Frag*>(w + b * 16 * l.pitch_in + k * 32);
            const Frag fu = *reinterpret_cast<const Frag*>(w + (32 + b * 16) * l.pitch_in + k * 32);
#pragma unroll
            for (int i = 0; i < RG; i++) {
              g[i][b] = Mma<T>::run(fg, x[i][k], g[i][b]);
              u[i][b] = Mma<T>::run(fu, x[i][k], u[i][b]);
            }
          }
        Frag h[RG];
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            float unused;
            float v = act_value<T, kAct, false>(g[i][e >> 2][e & 3], unused) * u[i][e >> 2][e & 3];
            if (kEnds && h0 + hc + q * 4 + (e & 3) + (e >> 2) * 16 >= p.hidden) v = 0.0f;
            h[i][e] = from_f32<T>(v);
          }
#pragma unroll
        for (int o = 0; o < FO; o++) {
          const Frag fd = *reinterpret_cast<const Frag*>(w_down + o * 16 * l.pitch_h + hc);
#pragma unroll
          for (int i = 0; i < RG; i++) y[i][o] = Mma<T>::run(fd, h[i], y[i][o]);
        }
      }
    }
    load_x(row + step);   // on its way while y is stored
    if (p.out % 8 == 0) {
#pragma unroll
      for (int i = 0; i < RG; i++)
        store_rows<T, FO>(stage, p.y, row + i * 16, p.rows, 0, p.out, [&](int j) { return y[i][j]; }, lane);
    } else {
#pragma unroll
      for (int i = 0; i < RG; i++)
#pragma unroll
        for (int o = 0; o < FO; o++)
          if (row + i * 16 + r < p.rows) store4(p.y + (row + i * 16 + r) * p.out, o * 16 + q * 4, p.out, false, y[i][o]);
    }
  }
}

template <typename T, int KI>
hipError_t narrow_forward(const Narrow<T>& p, hipStream_t s) {
  // 32 rows a wave: up to 64 features that leaves registers for four waves a SIMD, one's activation beside
  // another's products.  64 rows a wave and two waves: 145 us instead of 124 on 1,702,400 x 64, hidden 128 bf16.
  constexpr int RG = 2;
  const bool small = p.rows < (int64_t)256 * 8 * 16 * RG;   // fewer rows than a full chip's waves take: smaller workgroups
  const int waves = small ? 4 : 8, h32 = (p.hidden + 31) / 32 * 32;
  // hidden features in LDS at a time: all, or equal parts that fit
  int parts = 1, chunk = h32;
  while (narrow_lds(KI, chunk, waves).total * sizeof(T) > kNarrowLdsBytes) {
    parts++;
    chunk = (h32 / 32 + parts - 1) / parts * 32;
  }
  const int64_t tiles = (p.rows + 16 * RG * waves - 1) / (16 * RG * waves);
  const size_t lds = (size_t)narrow_lds(KI, chunk, waves).total * sizeof(T);
  const int64_t full = 256 * (lds <= 80 * 1024 ? 2 : 1);
  with_act(p.act, [&](auto act) {
    const unsigned grid = (unsigned)(tiles < full ? tiles : full);
    if (p.hidden % 32) narrow_forward_kernel<T, act.value, KI, RG, true><<<grid, waves * 64, lds, s>>>(p, chunk);
    else narrow_forward_kernel<T, act.value, KI, RG, false><<<grid, waves * 64, lds, s>>>(p, chunk);
  });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_narrow_forward(const GatedParams& g, hipStream_t s) {
  const Narrow<T> p{static_cast<const T*>(g.x), static_cast<const T*>(g.w_gate), static_cast<const T*>(g.w_up),
                    static_cast<const T*>(g.w_down), static_cast<T*>(g.y), g.rows, g.in, g.hidden, g.out, g.activation};
  const int side = g.in > g.out ? g.in : g.out;
  if (side <= 32) return narrow_forward<T, 1>(p, s);
  if (side <= 64) return narrow_forward<T, 2>(p, s);
  if (side <= 96) return narrow_forward<T, 3>(p, s);
  return narrow_forward<T, 4>(p, s);
}

// ---- backward ----
//
// One kernel makes g, u and dh again, dx, and the weight gradients' sums, so
// that a step reads x and dy and writes dx and nothing of the size of h.  A
// group of SL waves takes 32 rows at a time, wave s the hidden features
// 32 s .. 32 s + 31 of all of them; its share of the three weight gradients
// stays in its accumulators over all rows (96 registers for 64 features).
// dg, du and h go through LDS as [row][hidden]: read along a row they are
// operands of dx, whose sum over all hidden features is dealt out by its own
// columns; read transposed (32 rows as the product's k) they are operands of
// the weight gradients, as are x and dy.  One copy of the weights in LDS
// serves both directions for the same reason.
//
// Measured, 640,000 x 32, hidden 128 f16 with ReLU: 79 us and 4 to join the
// workgroups' sums; LDS busy 0.49 of the time, the vector ALU 0.48, the matrix
// cores 0.25: two waves a SIMD with two barriers a turn.  1,702,400 x 64, 128
// bf16 375 us.
//
// More hidden features than a group's waves have (256, or 128 for over 64
// features) take a launch each for equal parts of them; dx is summed between
// the launches in float32, in the order the accumulators hold it.

template <typename T>
struct NarrowBack {
  const T *x, *wg, *wu, *wd, *dy;
  T* dx;            // or null
  float* dx_sum;    // sums of dx between launches, see below
  float* part;      // [workgroups][dWg, dWu: slices 32 x in padded; dWd: out padded x slices 32]
  int64_t rows;
  int in, hidden, out, act;
  int first, last;  // hidden features of this launch
};

// Rows of n elements in LDS, n a power of two, their 16-byte chunks permuted by
// the row (its low four bits) such that none of the three ways they are touched
// meets a bank twice: 16-byte reads of 16 rows, transposing reads of rows 0 to 3
// and 8 to 11 at once, 8-byte writes of 16 rows.  Each is an address of the lane
// XOR a multiple of 16 columns, plus whole rows.
template <int n>
struct Rows {
  static __device__ __forceinline__ int permute(int row) {
    const int b0 = row & 1, b1 = row >> 1 & 1, b2 = row >> 2 & 1, b3 = row >> 3 & 1;
    if constexpr (n == 32) return b2 * 2 ^ b3 * 3;
    if constexpr (n == 64) return b1 * 2 ^ b2 * 4 ^ b3 * 5;
    return b0 * 2 ^ b1 * 4 ^ b2 * 8 ^ b3 * 9;
  }
  static __device__ __forceinline__ int at(int row, int col) { return row * n + (((col >> 3) ^ permute(row)) << 3) + (col & 7); }

  int along_, down_[2], put_;
  __device__ __forceinline__ Rows() {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    along_ = at(r, q * 8);
    down_[0] = at(q * 8 + (r >> 2), (r & 3) * 4);
    down_[1] = at(q * 8 + (r >> 2) + 4, (r & 3) * 4);
    put_ = at(r, q * 4);
  }
  // Hides the lane's addresses from the compiler, which would otherwise keep
  // every one of their XORs in registers over a loop.
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(along_), "+v"(down_[0]), "+v"(down_[1]), "+v"(put_)); }
  // Eight values along row `row` + lane % 16 from column `col` + 8 (lane / 16) on; row a multiple of 16, col of 32.
  template <typename T>
  __device__ __forceinline__ typename Mma<T>::Frag along(const T* p, int row, int col) const {
    return *reinterpret_cast<const typename Mma<T>::Frag*>(p + (along_ ^ col) + row * n);
  }
  // Eight values down column `col` + lane % 16 from row `row` + 8 (lane / 16) on; row a multiple of 32, col of 16.
  template <typename T>
  __device__ __forceinline__ typename Mma<T>::Frag down(const T* p, int row, int col) const {
    i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(p + (down_[0] ^ col) + row * n));
    i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(p + (down_[1] ^ col) + row * n));
    return __builtin_bit_cast(typename Mma<T>::Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // Four values at row `row` + lane % 16, column `col` + 4 (lane / 16).
  template <typename T>
  __device__ __forceinline__ void put(T* p, int row, int col, const Four<T>& v) const {
    *reinterpret_cast<Four<T>*>(p + (put_ ^ col) + row * n) = v;
  }
};

// kEnds: the launch's hidden features end before its slices do.  dx sums over
// all of them: dg and du past the last one are zero, where an infinity times
// its weights of zero would make the row NaN.
template <typename T, int KI, int SL, bool kEnds>
__global__ __launch_bounds__(64 * narrow_back_waves(KI), KI <= 2 ? 2 : 1) void narrow_backward_kernel(NarrowBack<T> p) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int kWaves = narrow_back_waves(KI), kGroups = kWaves / SL, kThreads = 64 * kWaves;
  constexpr NarrowBackLds l = narrow_back_lds(KI, SL);
  constexpr int H = SL * 32, PI = l.row_in, PH = l.row_h, FI = 2 * KI;
  typedef Rows<PI> In;
  typedef Rows<PH> Hid;
  In in;
  Hid hid;
  static_assert(l.groups == kGroups, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t narrow_mem[];
  T* const lds = reinterpret_cast<T*>(narrow_mem);
  T *const wg = lds, *const wu = lds + H * PI, *const wd = lds + 2 * H * PI;
  for (int c = threadIdx.x; c < 2 * H * KI * 4; c += kThreads) {
    const int row = c / (KI * 4), k = c % (KI * 4) * 8, h = row < H ? row : row - H;
    *reinterpret_cast<Frag*>((row < H ? wg : wu) + In::at(h, k)) =
        load8<T>((row < H ? p.wg : p.wu) + (int64_t)(p.first + h) * p.in + k, p.first + h < p.last ? p.in - k : 0);
  }
  for (int c = threadIdx.x; c < KI * 32 * (H / 8); c += kThreads) {
    const int o = c / (H / 8), k = c % (H / 8) * 8, h = p.first + k;
    *reinterpret_cast<Frag*>(wd + Hid::at(o, k)) = load8<T>(p.wd + (int64_t)o * p.hidden + h, o < p.out ? p.last - h : 0);
  }
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int group = wave_id() / SL, slice = wave_id() % SL, t = threadIdx.x % (SL * 64);
  T* const xs = lds + l.tiles + group * l.tile_stride;
  T* const dys = xs + 32 * PI;
  T* const dg = dys + 32 * PI;
  T* const du = dg + 32 * PH;
  // x and dy of the next rows, in registers until their place in LDS is free
  constexpr int kChunks = 256 * KI, kLoads = (kChunks + SL * 64 - 1) / (SL * 64);
  Frag next[kLoads];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int c = t + i * SL * 64, half = c / (kChunks / 2), e = c % (kChunks / 2);
      const int64_t n = row + e / (KI * 4);
      const int k = e % (KI * 4) * 8, len = half ? p.out : p.in;
      next[i] = load8<T>((half ? p.dy : p.x) + n * len + k, c < kChunks && n < p.rows ? len - k : 0);
    }
  };
  auto place = [&]() {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int c = t + i * SL * 64, half = c / (kChunks / 2), e = c % (kChunks / 2);
      if (c < kChunks) *reinterpret_cast<Frag*>((half ? dys : xs) + In::at(e / (KI * 4), e % (KI * 4) * 8)) = next[i];
    }
  };
  f32x4 dwg[2][FI] = {}, dwu[2][FI] = {}, dwd[FI][2] = {};
  // every group of the workgroup takes the same number of turns: barriers stand inside
  const int64_t first = ((int64_t)blockIdx.x * kGroups) * 32, step = (int64_t)gridDim.x * kGroups * 32;
  load(first + group * 32);
  place();
  __syncthreads();
  for (int64_t base = first; base < p.rows; base += step) {
    const int64_t row = base + group * 32;
    in.renew();
    hid.renew();
    load(row + step);
    f32x4 g[2][2] = {}, u[2][2] = {}, dh[2][2] = {};   // [16 hidden][16 rows]
#pragma unroll
    for (int k = 0; k < KI; k++) {
      Frag fx[2], fy[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        fx[i] = in.along(xs, i * 16, k * 32);
        fy[i] = in.along(dys, i * 16, k * 32);
      }
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int h = slice * 32 + b * 16;
        const Frag fg = in.along(wg, h, k * 32), fu = in.along(wu, h, k * 32), fd = hid.down(wd, k * 32, h);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          g[b][i] = Mma<T>::run(fg, fx[i], g[b][i]);
          u[b][i] = Mma<T>::run(fu, fx[i], u[b][i]);
          dh[b][i] = Mma<T>::run(fd, fy[i], dh[b][i]);
        }
      }
    }
    // dg, du and h of this wave's own columns, which no other wave reads before
    // the barrier: h first takes dg's place to be read transposed
    Four<T> vg[2][2], vu[2][2], vh[2][2];
    with_act(p.act, [&](auto act) {
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float slope;
            const float a = act_value<T, act.value, true>(g[b][i][e], slope), d = dh[b][i][e];
            vg[b][i].v[e] = from_f32<T>(d * u[b][i][e] * slope);
            vu[b][i].v[e] = from_f32<T>(d * a);
            vh[b][i].v[e] = from_f32<T>(a * u[b][i][e]);
          }
    });
    if constexpr (kEnds) {
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (p.first + slice * 32 + b * 16 + q * 4 + e >= p.last)
            vg[b][0].v[e] = vg[b][1].v[e] = vu[b][0].v[e] = vu[b][1].v[e] = (T)0.0f;
    }
    auto put = [&](T* to, const Four<T> (&v)[2][2]) {
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 2; i++) hid.put(to, i * 16, slice * 32 + b * 16, v[b][i]);
    };
    auto settle = [&]() {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    put(dg, vh);
    put(du, vu);
    settle();
    {
      Frag fh[2];
#pragma unroll
      for (int b = 0; b < 2; b++) fh[b] = hid.down(dg, 0, slice * 32 + b * 16);
#pragma unroll
      for (int j = 0; j < FI; j++) {
        const Frag fy = in.down(dys, 0, j * 16);
#pragma unroll
        for (int b = 0; b < 2; b++) dwd[j][b] = Mma<T>::run(fy, fh[b], dwd[j][b]);
      }
    }
    settle();
    put(dg, vg);
    settle();
    {
      Frag fg[2], fu[2];
#pragma unroll
      for (int b = 0; b < 2; b++) {
        fg[b] = hid.down(dg, 0, slice * 32 + b * 16);
        fu[b] = hid.down(du, 0, slice * 32 + b * 16);
      }
#pragma unroll
      for (int j = 0; j < FI; j++) {
        const Frag fx = in.down(xs, 0, j * 16);
#pragma unroll
        for (int b = 0; b < 2; b++) {
          dwg[b][j] = Mma<T>::run(fg[b], fx, dwg[b][j]);
          dwu[b][j] = Mma<T>::run(fu[b], fx, dwu[b][j]);
        }
      }
    }
    __syncthreads();   // dg and du are whole; x and dy are no longer read
    place();
    if (p.dx && row < p.rows) {   // the whole group, and no barrier inside
      for (int tile = slice; tile < FI * 2; tile += SL) {
        const int j = tile >> 1, i = tile & 1;
        float* const sum = p.dx_sum + (((row >> 4) + i) * FI + j) * 256 + lane * 4;   // rows in whole 32s
        f32x4 acc = {};
        if (p.first) acc = *reinterpret_cast<const f32x4*>(sum);
#pragma unroll
        for (int k = 0; k < SL; k++) {
          acc = Mma<T>::run(in.down(wg, k * 32, j * 16), hid.along(dg, i * 16, k * 32), acc);
          acc = Mma<T>::run(in.down(wu, k * 32, j * 16), hid.along(du, i * 16, k * 32), acc);
        }
        const int64_t n = row + i * 16 + r;
        if (p.last < p.hidden) *reinterpret_cast<f32x4*>(sum) = acc;
        else if (n < p.rows) store4(p.dx + n * p.in, j * 16 + q * 4, p.in, p.in % 4 == 0, acc);
      }
    }
    __syncthreads();   // the next x and dy are whole; dg and du are no longer read
  }
  // the groups' sums, in their order, through the LDS that the weights had
  int last_lane = threadIdx.x & 63;
  asm volatile("" : "+v"(last_lane));   // made again here, not held in a register over the rows
  f32x4* const sums = reinterpret_cast<f32x4*>(narrow_mem) + slice * (6 * FI * 64) + last_lane;
  for (int other = 1; other < kGroups; other++) {
    if (group == other) {
#pragma unroll
      for (int j = 0; j < FI; j++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          sums[((j * 2 + b) * 3 + 0) * 64] = dwg[b][j];
          sums[((j * 2 + b) * 3 + 1) * 64] = dwu[b][j];
          sums[((j * 2 + b) * 3 + 2) * 64] = dwd[j][b];
        }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < FI; j++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          dwg[b][j] += sums[((j * 2 + b) * 3 + 0) * 64];
          dwu[b][j] += sums[((j * 2 + b) * 3 + 1) * 64];
          dwd[j][b] += sums[((j * 2 + b) * 3 + 2) * 64];
        }
    }
    __syncthreads();
  }
  if (group != 0) return;
  constexpr int D = KI * 32;
  float* const part = p.part + (int64_t)blockIdx.x * (3 * H * D);
#pragma unroll
  for (int j = 0; j < FI; j++)
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int row4 = (last_lane >> 4) * 4 + e, col = last_lane & 15, h = slice * 32 + b * 16 + row4;
        part[h * D + j * 16 + col] = dwg[b][j][e];
        part[H * D + h * D + j * 16 + col] = dwu[b][j][e];
        part[2 * H * D + (j * 16 + row4) * H + slice * 32 + b * 16 + col] = dwd[j][b][e];
      }
}

// The weight gradients from the workgroups' sums: 32 places a workgroup, 32
// slices of the sums, joined in LDS in a fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void narrow_join_kernel(const float* part, int n, int H, int D, int in, int hidden, int out,
                                                           int first, int last, T* dwg, T* dwu, T* dwd) {
  __shared__ float lds[32][33];
  const int size = 3 * H * D, col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float s = 0.0f;
  for (int i = slice; i < n; i += 32) s += part[(int64_t)i * size + col];   // size is a multiple of 32
  lds[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice) return;
  float v = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; i++) v += lds[i][threadIdx.x];
  const int which = col / (H * D), e = col % (H * D);
  if (which < 2) {
    T* to = which ? dwu : dwg;
    const int h = first + e / D, i = e % D;
    if (to && h < last && i < in) to[(int64_t)h * in + i] = from_f32<T>(v);
  } else {
    const int o = e / H, h = first + e % H;
    if (dwd && o < out && h < last) dwd[(int64_t)o * hidden + h] = from_f32<T>(v);
  }
}

template <typename T, int KI, int SL>
hipError_t narrow_backward(const GatedParams& g, const GatedLayout& l, hipStream_t s) {
  constexpr NarrowBackLds m = narrow_back_lds(KI, SL);
  uint8_t* const ws = static_cast<uint8_t*>(g.ws);
  const int per = (g.hidden + l.narrow_parts - 1) / l.narrow_parts;
  for (int first = 0; first < g.hidden; first += per) {
    const int last = first + per < g.hidden ? first + per : g.hidden;
    const NarrowBack<T> p{static_cast<const T*>(g.x), static_cast<const T*>(g.w_gate), static_cast<const T*>(g.w_up),
                          static_cast<const T*>(g.w_down), static_cast<const T*>(g.dy), static_cast<T*>(g.dx),
                          reinterpret_cast<float*>(ws + l.dx_sum), reinterpret_cast<float*>(ws + l.part), g.rows, g.in, g.hidden, g.out,
                          g.activation, first, last};
    constexpr int H = SL * 32, D = KI * 32;
    if (last - first < H) narrow_backward_kernel<T, KI, SL, true><<<l.narrow_groups, 64 * narrow_back_waves(KI), m.total * sizeof(T), s>>>(p);
    else narrow_backward_kernel<T, KI, SL, false><<<l.narrow_groups, 64 * narrow_back_waves(KI), m.total * sizeof(T), s>>>(p);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (g.dw_gate || g.dw_up || g.dw_down)
      narrow_join_kernel<T><<<3 * H * D / 32, 1024, 0, s>>>(p.part, l.narrow_groups, H, D, g.in, g.hidden, g.out, first, last,
                                                            static_cast<T*>(g.dw_gate), static_cast<T*>(g.dw_up), static_cast<T*>(g.dw_down));
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int KI>
hipError_t narrow_backward_slices(const GatedParams& g, const GatedLayout& l, hipStream_t s) {
  const int slices = l.narrow_slices;
  if constexpr (KI != 2)
    if (slices == 1) return narrow_backward<T, KI, 1>(g, l, s);
  if (slices == 2) return narrow_backward<T, KI, 2>(g, l, s);
  if constexpr (KI <= 2)
    if (slices == 8) return narrow_backward<T, KI, 8>(g, l, s);
  return narrow_backward<T, KI, 4>(g, l, s);
}

template <typename T>
hipError_t launch_narrow_backward(const GatedParams& g, const GatedLayout& l, hipStream_t s) {
  const int side = g.in > g.out ? g.in : g.out;
  if (side <= 32) return narrow_backward_slices<T, 1>(g, l, s);
  if (side <= 64) return narrow_backward_slices<T, 2>(g, l, s);
  if (side <= 96) return narrow_backward_slices<T, 3>(g, l, s);
  return narrow_backward_slices<T, 4>(g, l, s);
}

}  // namespace
}  // namespace nest
