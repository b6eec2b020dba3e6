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

template <typename T, int kAct, int KI, int RG>
__global__ __launch_bounds__(512, 2) void narrow_forward_kernel(Narrow<T> p) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int FO = 2 * KI;
  extern __shared__ __attribute__((aligned(16))) uint8_t narrow_mem[];
  T* lds = reinterpret_cast<T*>(narrow_mem);
  const int waves = blockDim.x >> 6;
  const NarrowLds l = narrow_lds(KI, p.hidden, waves);
  const int h32 = (p.hidden + 31) & ~31;
  // weights; what lies past a matrix is zero
  for (int c = threadIdx.x; c < 2 * h32 * (KI * 4); c += blockDim.x) {
    const int row = c / (KI * 4), k = c % (KI * 4) * 8;
    const int h = (row >> 6) * 32 + (row & 31);
    const T* w = row & 32 ? p.wu : p.wg;
    const Frag f = load8<T>(w + (int64_t)h * p.in + k, h < p.hidden ? p.in - k : 0);
    *reinterpret_cast<Frag*>(lds + row * l.pitch_in + k) = f;
  }
  for (int c = threadIdx.x; c < KI * 32 * (h32 / 8); c += blockDim.x) {
    const int o = c / (h32 / 8), k = c % (h32 / 8) * 8;   // elements k .. k + 7 of a row in LDS: a chunk's quarter
    const int base = (k & ~31) + ((k >> 3) & 3) * 4;
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int h = base + (e & 3) + (e >> 2) * 16;
      f[e] = o < p.out && h < p.hidden ? p.wd[(int64_t)o * p.hidden + h] : (T)0.0f;
    }
    *reinterpret_cast<Frag*>(lds + l.down + o * l.pitch_h + k) = f;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const T* w_in = lds + r * l.pitch_in + q * 8;
  const T* w_down = lds + l.down + r * l.pitch_h + q * 8;
  auto& stage = *reinterpret_cast<RowStage<T, FO>*>(lds + l.stage + wave_id() * 16 * RowStage<T, FO>::kPitch);
  const int64_t step = (int64_t)gridDim.x * waves * (16 * RG);
  int64_t row = ((int64_t)blockIdx.x * waves + wave_id()) * (16 * RG);
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
  if (row < p.rows) load_x(row);
  for (; row < p.rows; row += step) {
    f32x4 y[RG][FO] = {};
    for (int hc = 0; hc < h32; hc += 32) {
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
          h[i][e] = from_f32<T>(act_value<T, kAct, false>(g[i][e >> 2][e & 3], unused) * u[i][e >> 2][e & 3]);
        }
#pragma unroll
      for (int o = 0; o < FO; o++) {
        const Frag fd = *reinterpret_cast<const Frag*>(w_down + o * 16 * l.pitch_h + hc);
#pragma unroll
        for (int i = 0; i < RG; i++) y[i][o] = Mma<T>::run(fd, h[i], y[i][o]);
      }
    }
    if (row + step < p.rows) load_x(row + step);   // on its way while y is stored
    if (p.out % 8 == 0) {
#pragma unroll
      for (int i = 0; i < RG; i++)
        store_rows<T, FO>(stage, p.y, row + i * 16, p.rows, 0, p.out, [&](int j) { return y[i][j]; });
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
  // 64 rows a wave where registers allow: each weight fragment read from LDS is used RG times
  constexpr int RG = KI <= 2 ? 4 : 2;
  const bool small = p.rows < (int64_t)256 * 8 * 16 * RG;   // fewer rows than a full chip's waves take: smaller workgroups
  const int waves = small ? 4 : 8;
  const int64_t tiles = (p.rows + 16 * RG * waves - 1) / (16 * RG * waves);
  const size_t lds = (size_t)narrow_lds(KI, p.hidden, waves).total * sizeof(T);
  const int64_t full = 256 * (lds <= 80 * 1024 ? 2 : 1);
  with_act(p.act, [&](auto act) {
    narrow_forward_kernel<T, act.value, KI, RG><<<(unsigned)(tiles < full ? tiles : full), waves * 64, lds, s>>>(p);
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

}  // namespace
}  // namespace nest
