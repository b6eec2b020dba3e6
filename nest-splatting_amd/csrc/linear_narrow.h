// The dense layer for narrow rows (at most 128 features in and out) of a
// 16-bit type: whole rows stay in registers, the weights in LDS.
//
// A frame has a million rows of 16 to 128 features, so a forward is bound by
// reading x and the residual and writing y, a backward by reading x and dy and
// writing dx, and nothing of the rows' size is kept between the two: the
// backward makes z again from x, which it reads anyway, where the tiles would
// write and read two bytes of slope an element (a third of the traffic).  Only
// what is kept in 8 bits on request is read instead.
//
// A wave takes 16 or 32 rows.  It computes transposed products, weights as the first
// operand and rows as the second, with the first operand's rows in an order by
// which a lane's accumulators of two fragments are 8 consecutive features of
// one row: 16 bytes of y, of dy, or of the second operand of the next product,
// so no value changes lanes between loads, products and stores.  The weights'
// gradient sums over rows: the four waves of a workgroup put dz and x into LDS
// and each takes a part of the gradient over a turn's 64 rows with transposing
// reads; it gathers in registers over the turns.
//
// 1,702,400 x 64 -> 64 of bf16 with GELU and a residual: forward 139 us (654 MB:
// 4.7 TB/s, the vector ALU 0.61 busy with the exponential and reciprocal of
// every result), backward 167 (654 MB: 3.9 TB/s; vector ALU 0.62, LDS 0.43, of
// which conflicts 0.20).  us of a forward and a backward here and in tiles:
// 640,000 x 64 -> 64 37 + 61 and 56 + 129, 32 -> 128 63 + 97 and 130 + 194, 128
// -> 128 89 + 224 and 161 + 262, with 8 bits 89 + 180 and 149 + 248; 16,384 rows
// of 128 -> 128 11 + 27 and 13 + 30, 64 rows 12 + 21 and 15 + 28.  float32 has
// kernels of its own (linear_narrow_f32.h).
#pragma once

#include "linear_tiles.h"

namespace nest {
namespace {

// Groups of 16 rows that a wave takes in a turn: two share a read of the
// weights.
constexpr int forward_groups(int ki, int ko) { return ki + ko <= 4 ? 2 : 1; }

template <typename T>
struct NarrowLayer {
  const T *x, *w, *bias;     // a backward's x may be null: codes hold it, or nothing asks for it
  const int8_t* codes;       // x in 8 bits, or null
  const uint8_t* steps;
  int64_t rows;
  int in, out, act;
  const T* residual;         // forward; or null
  T* y;
  uint8_t* kept;
  const T* dy;               // backward
  const uint8_t* slopes;     // or null: none, or made again
  T* dx;
  float *dw, *db;            // [groups][out][in], [groups][out]; each may be null
};

// 16 bytes of a row as a fragment.  What a loop carries stays words: the
// compiler would take a register for each element of a fragment.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag frag_of(const Words16<T>& w) {
  return __builtin_bit_cast(typename Mma<T>::Frag, w);
}

// 8 bytes of a row with n left at p, zeros past its end.
__device__ __forceinline__ uint2 row_bytes(const void* p, int n) {
  uint2 v = make_uint2(0, 0);
  if (n >= 8) {
    __builtin_memcpy(&v, p, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) (i < 4 ? v.x : v.y) |= (uint32_t)static_cast<const uint8_t*>(p)[i] << (i % 4 * 8);
  }
  return v;
}
__device__ __forceinline__ void store_bytes(uint8_t* p, uint2 v, int n) {
  if (n >= 8) {
    store_whole(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) p[i] = (uint8_t)((i < 4 ? v.x : v.y) >> (i % 4 * 8));
  }
}
__device__ __forceinline__ float byte_of(uint2 v, int i) { return (float)(((i < 4 ? v.x : v.y) >> (i % 4 * 8)) & 0xffu); }

// A [rows][cols] matrix of the weights (transposed: [cols][rows] in memory) to
// LDS, zeros around it, its rows in the order that the products read them:
// pitches of an odd number of 16 bytes, so 16 rows one after another fall on
// different banks.
template <typename T, int R, int C, bool kTransposed>
__device__ __forceinline__ void stage_weights(T* lds, const T* w, int rows, int cols) {
  constexpr int kPitch = C + 8, kLong = kTransposed ? R : C;   // of a row in memory
  constexpr int kPieces = (R * C + 8 * 256 - 1) / (8 * 256);   // of 16 bytes, a thread's
  const int length = kTransposed ? rows : cols, lines = kTransposed ? cols : rows;
  Words16<T> v[kPieces];   // all on their way at once: one after another takes 20 us
#pragma unroll
  for (int u = 0; u < kPieces; u++) {
    const int i = (u * 256 + threadIdx.x) * 8, line = i / kLong, at = i % kLong;
    v[u] = load_words<false>(w + line * length + at, line < lines ? length - at : 0);
  }
#pragma unroll
  for (int u = 0; u < kPieces; u++) {
    const int i = (u * 256 + threadIdx.x) * 8, line = i / kLong, at = i % kLong;
    if (i >= R * C) break;
    auto row_at = [](int r) { return ((r & ~31) | (r >> 2 & 1) << 4 | (r >> 3 & 3) << 2 | (r & 3)) * kPitch; };
    if constexpr (kTransposed) {
#pragma unroll
      for (int e = 0; e < 8; e++) lds[row_at(at + e) + line] = v[u][e];
    } else {
      *reinterpret_cast<uint4*>(lds + row_at(line) + at) = __builtin_bit_cast(uint4, v[u]);
    }
  }
}

// acc[jj][g] over K / 32 steps, from init on: features 32 J + 8 (lane / 16) +
// 4 jj + 0..3 of row lane % 16 of group g.  Row m of the first operand in half
// jj of 32 is feature 8 (m / 4) + m % 4 + 4 jj.
template <typename T, int K, int G>
__device__ __forceinline__ void narrow_product(const T* lds, int J, const typename Mma<T>::Frag (&rows)[G][K / 32], const f32x4 (&init)[2],
                                               f32x4 (&acc)[2][G]) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int jj = 0; jj < 2; jj++)
#pragma unroll
    for (int g = 0; g < G; g++) acc[jj][g] = init[jj];
#pragma unroll
  for (int k = 0; k < K / 32; k++)
#pragma unroll
    for (int jj = 0; jj < 2; jj++) {
      const auto a = *reinterpret_cast<const typename Mma<T>::Frag*>(lds + (32 * J + 16 * jj + r) * (K + 8) + k * 32 + q * 8);
#pragma unroll
      for (int g = 0; g < G; g++) acc[jj][g] = Mma<T>::run(a, rows[g][k], acc[jj][g]);
    }
}

// The bias to LDS, zeros after it: float32, four to an element.
template <typename T>
__device__ __forceinline__ void stage_bias(f32x4* lds, const T* bias, int out, int padded) {
  for (int i = threadIdx.x; i < padded; i += 256) reinterpret_cast<float*>(lds)[i] = bias && i < out ? to_f32(bias[i]) : 0.0f;
}

// Row of 16 in LDS, in 8 bytes.
template <int KO>
constexpr int kCodePitch = KO * 4 + 2;

// kKept: the slopes' codes are written too, a row's side by side through LDS: a
// wave's own, eight bytes a lane, are 32 bytes of each of 16 rows, and memory
// took 46% more requests for them than their bytes need.
template <typename T, int KI, int KO, bool kKept>
__global__ __launch_bounds__(256, 3) void narrow_layer_kernel(NarrowLayer<T> p) {
  typedef typename Mma<T>::Frag Frag;
  __shared__ __attribute__((aligned(16))) T w[KO * 32 * (KI * 32 + 8)];
  __shared__ f32x4 bias[KO * 8];
  __shared__ __attribute__((aligned(16))) uint2 codes[kKept ? 4 : 1][kKept ? 16 * kCodePitch<KO> : 1];   // of a wave's 16 rows
  stage_weights<T, KO * 32, KI * 32, false>(w, p.w, p.out, p.in);
  stage_bias(bias, p.bias, p.out, KO * 32);
  __syncthreads();
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  constexpr int G = forward_groups(KI, KO);
  const int64_t step = (int64_t)gridDim.x * 64 * G;
  Words16<T> x[G][KI], res[G][KO];
  auto load = [&](int64_t at) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      const bool in = at + g * 16 < p.rows;
#pragma unroll
      for (int k = 0; k < KI; k++) x[g][k] = load_words<false>(p.x + (at + g * 16) * p.in + k * 32 + q * 8, in ? p.in - k * 32 - q * 8 : 0);
      if (p.residual) {
#pragma unroll
        for (int k = 0; k < KO; k++) res[g][k] = load_words<false>(p.residual + (at + g * 16) * p.out + k * 32 + q * 8, in ? p.out - k * 32 - q * 8 : 0);
      }
    }
  };
  int64_t row = ((int64_t)blockIdx.x * 4 + wave_id()) * 16 * G + r;
  load(row);
  for (; row - r < p.rows; row += step) {
    Frag now[G][KI];
    Words16<T> add[G][KO];
#pragma unroll
    for (int g = 0; g < G; g++) {
#pragma unroll
      for (int k = 0; k < KI; k++) now[g][k] = frag_of(x[g][k]);
#pragma unroll
      for (int k = 0; k < KO; k++) add[g][k] = res[g][k];
    }
    load(row + step);   // on its way while this turn is worked on
    uint2 mine[G][kKept ? KO : 1];
#pragma unroll
    for (int J = 0; J < KO; J++) {
      const f32x4 init[2] = {bias[J * 8 + q * 2], bias[J * 8 + q * 2 + 1]};
      f32x4 acc[2][G];
      narrow_product<T, KI * 32, G>(w, J, now, init, acc);
      const int c = J * 32 + q * 8;
#pragma unroll
      for (int g = 0; g < G; g++) {
        float v[8];
        uint2 code = make_uint2(0, 0);
        with_activation(p.act, [&](auto act) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            float slope;
            v[e] = activate<T, act.value, kKept>(acc[e >> 2][g][e & 3], slope);
            if constexpr (kKept) (e < 4 ? code.x : code.y) |= (uint32_t)coarse_code(slope) << (e % 4 * 8);
          }
        });
        if constexpr (kKept) mine[g][J] = code;
        if (p.residual) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] += to_f32(add[g][J][e]);
        }
        store_vec<T>(p.y + (row + g * 16) * p.out + c, v, row + g * 16 < p.rows ? p.out - c : 0);
      }
      __builtin_amdgcn_sched_barrier(0);   // one 32 features at a time: their registers are the next one's
    }
    if constexpr (kKept) {
      uint2* const stage = codes[wave_id()];
#pragma unroll
      for (int g = 0; g < G; g++) {
#pragma unroll
        for (int J = 0; J < KO; J++) stage[r * kCodePitch<KO> + J * 4 + q] = mine[g][J];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < (KO + 1) / 2; u++) {   // 16 bytes: KO * 2 to a row
          const int t = u * 64 + lane, at = t / (KO * 2), c = t % (KO * 2) * 16;
          const int64_t to = row - r + g * 16 + at;
          if (at < 16 && to < p.rows) {
            const uint4 v = *reinterpret_cast<const uint4*>(&stage[at * kCodePitch<KO> + c / 8]);
            uint8_t* const y = p.kept + to * p.out + c;
            store_bytes(y, make_uint2(v.x, v.y), p.out - c);
            store_bytes(y + 8, make_uint2(v.z, v.w), p.out - c - 8);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

constexpr int pow2_of(int k) { return k == 3 ? 4 : k; }   // 32s of a tile's row

// LDS of the backward, in elements.
template <int KI, int KO, bool kSaved>
struct NarrowLayerLds {
  static constexpr int rows = kNarrowBackRows;
  static constexpr int RO = pow2_of(KO) * 32, RI = pow2_of(KI) * 32;
  static constexpr int wt = kSaved ? 0 : KO * 32 * (KI * 32 + 8);
  static constexpr int dz = wt + KI * 32 * (KO * 32 + 8);
  static constexpr int x = dz + rows * RO;
  static constexpr int total = x + rows * RI;
};

// Where a lane's 8 elements of a row go in a tile of R columns that is read
// transposed (tile_gemm.h).
template <typename T, int R>
__device__ __forceinline__ int tile_place(int row, int J, int q) {
  return row * R + (((2 * J + (q >> 1)) ^ unit_swizzle<T, R>(row)) << 4) + (q & 1) * 8;
}

// kSaved: what the backward needs may lie in 8 bits, x (codes) as well as the
// slopes, and no slopes are made again.
template <typename T, int KI, int KO, bool kSaved>
__global__ __launch_bounds__(256, narrow_groups_cu(KI, KO, kSaved)) void narrow_layer_backward_kernel(NarrowLayer<T> p) {
  typedef typename Mma<T>::Frag Frag;
  typedef NarrowLayerLds<KI, KO, kSaved> L;
  constexpr int G = 1, kRows = L::rows, NO = 2 * KO, NI = 2 * KI;
  constexpr int WO = NO % 4 == 0 ? 4 : 2, WI = 4 / WO, FO = NO / WO, FI = NI / WI;   // waves and fragments of dW
  __shared__ __attribute__((aligned(16))) T lds[L::total];
  __shared__ f32x4 bias[kSaved ? 1 : KO * 8];
  const bool again = !kSaved && p.act != NEST_ACT_NONE;   // w may be null without it and dx
  if constexpr (!kSaved) {
    if (again) {
      stage_bias(bias, p.bias, p.out, KO * 32);
      stage_weights<T, KO * 32, KI * 32, false>(lds, p.w, p.out, p.in);
    }
  }
  if (p.dx) stage_weights<T, KI * 32, KO * 32, true>(lds + L::wt, p.w, p.in, p.out);
  __syncthreads();
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = wave_id();
  const int64_t step = (int64_t)gridDim.x * kRows;
  const int64_t first = (int64_t)blockIdx.x * kRows;
  Words16<T> xw[G][KI], dy[G][KO];
  uint2 slopes[G][KO], codes[G][KI];
  int steps[G][KI];
  const int groups_in = (p.in + 31) / 32;
  auto load = [&](int64_t turn) {   // branches around the loops: inside, each load would wait for the last
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int64_t at = turn + wave * 16 * G + g * 16 + r;
      const bool in = at < p.rows;
      auto left = [&](int k, int cols) { return in ? cols - k * 32 - q * 8 : 0; };
      auto place = [&](int k, int cols) { return at * cols + k * 32 + q * 8; };
#pragma unroll
      for (int k = 0; k < KO; k++) dy[g][k] = load_words<false>(p.dy + place(k, p.out), left(k, p.out));
      if (kSaved && p.codes) {
#pragma unroll
        for (int k = 0; k < KI; k++) {
          codes[g][k] = row_bytes(p.codes + place(k, p.in), left(k, p.in));
          steps[g][k] = left(k, p.in) > 0 ? p.steps[at * groups_in + k] : 0;
        }
      } else {
#pragma unroll
        for (int k = 0; k < KI; k++) xw[g][k] = load_words<false>(p.x + place(k, p.in), p.x ? left(k, p.in) : 0);
      }
      if constexpr (kSaved) {
        if (p.slopes) {
#pragma unroll
          for (int k = 0; k < KO; k++) slopes[g][k] = row_bytes(p.slopes + place(k, p.out), left(k, p.out));
        }
      }
    }
  };
  load(first);
  f32x4 dw[FO][FI] = {};
  float db[KO][8] = {};
  const int wo = wave % WO, wi = wave / WO;
  const int base_o = fragment_base<T, false, L::RO>(0), base_i = fragment_base<T, false, L::RI>(0);
  for (int64_t turn = first; turn < p.rows; turn += step) {
    Frag x[G][KI], dz[G][KO];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int k = 0; k < KI; k++) x[g][k] = frag_of(xw[g][k]);
    if constexpr (kSaved) {
      if (p.codes) {
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int k = 0; k < KI; k++) {
            // a code and 128 as an unsigned byte; what lies past the row's end is of no gradient that is stored
            const uint2 c = make_uint2(codes[g][k].x ^ 0x80808080u, codes[g][k].y ^ 0x80808080u);
            const float step = steps[g][k] == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.0f, steps[g][k] - 132);
#pragma unroll
            for (int e = 0; e < 8; e++) x[g][k][e] = from_f32<T>((byte_of(c, e) - 128.0f) * step);
          }
      }
    }
#pragma unroll
    for (int J = 0; J < KO; J++) {
      float z[G][8];
      if (again) {
        const f32x4 init[2] = {bias[J * 8 + q * 2], bias[J * 8 + q * 2 + 1]};
        f32x4 acc[2][G];
        narrow_product<T, KI * 32, G>(lds, J, x, init, acc);
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int e = 0; e < 8; e++) z[g][e] = acc[e >> 2][g][e & 3];
        with_act(p.act, [&](auto act) {
#pragma unroll
          for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) activate<T, act.value>(z[g][e], z[g][e]);   // the slope in its place
        });
        if (J == KO - 1 && p.out % 32) {   // of no feature: an infinity in x makes its z NaN
#pragma unroll
          for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) z[g][e] = J * 32 + q * 8 + e < p.out ? z[g][e] : 0.0f;
        }
      }
      auto make_dz = [&](auto slope) {
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float d = to_f32(dy[g][J][e]) * slope(g, e);   // zero past the ends
            dz[g][J][e] = from_f32<T>(d);
            db[J][e] += d;
          }
      };
      if (kSaved && p.slopes) make_dz([&](int g, int e) { return coarse_slope(byte_of(slopes[g][J], e)); });
      else if (again) make_dz([&](int g, int e) { return z[g][e]; });
      else make_dz([&](int, int) { return 1.0f; });
      __builtin_amdgcn_sched_barrier(0);   // phases one after another: their registers are the next one's
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int at = wave * 16 * G + g * 16 + r;
#pragma unroll
      for (int k = 0; k < KO; k++) *reinterpret_cast<Frag*>(lds + L::dz + tile_place<T, L::RO>(at, k, q)) = dz[g][k];
#pragma unroll
      for (int k = 0; k < KI; k++) *reinterpret_cast<Frag*>(lds + L::x + tile_place<T, L::RI>(at, k, q)) = x[g][k];
    }
    load(turn + step);   // on its way while this turn is worked on
    if (p.dx) {
#pragma unroll
      for (int J = 0; J < KI; J++) {
        f32x4 acc[2][G];
        const f32x4 zero[2] = {};
        narrow_product<T, KO * 32, G>(lds + L::wt, J, dz, zero, acc);
        const int c = J * 32 + q * 8;
#pragma unroll
        for (int g = 0; g < G; g++) {
          const int64_t at = turn + wave * 16 * G + g * 16 + r;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = acc[e >> 2][g][e & 3];
          store_vec<T>(p.dx + at * p.in + c, v, at < p.rows ? p.in - c : 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();   // all rows of the turn are in LDS
    if (p.dw) {
      const uint8_t *tz = reinterpret_cast<const uint8_t*>(lds + L::dz), *tx = reinterpret_cast<const uint8_t*>(lds + L::x);
#pragma unroll
      for (int kb = 0; kb < kRows / 32; kb++) {
        Frag a[FO];
#pragma unroll
        for (int i = 0; i < FO; i++) a[i] = fragment<T, false, L::RO>(tz, base_o, wo * FO + i, kb);
#pragma unroll
        for (int j = 0; j < FI; j++) {
          const Frag b = fragment<T, false, L::RI>(tx, base_i, wi * FI + j, kb);
#pragma unroll
          for (int i = 0; i < FO; i++) dw[i][j] = Mma<T>::run(b, a[i], dw[i][j]);
        }
        if (kb % 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();   // and read
  }
  if (p.dw) {
    float* const part = p.dw + (int64_t)blockIdx.x * p.out * p.in;
#pragma unroll
    for (int i = 0; i < FO; i++)
#pragma unroll
      for (int j = 0; j < FI; j++) {
        const int o = (wo * FO + i) * 16 + r, c = (wi * FI + j) * 16 + q * 4;
        if (o < p.out) store4(part + o * p.in, c, p.in, p.in % 4 == 0, dw[i][j]);
      }
  }
  if (p.db) {
    float* const sums = reinterpret_cast<float*>(lds + L::dz);   // [4][KO * 32]
#pragma unroll
    for (int k = 0; k < KO; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float s = db[k][e];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
        if (r == 0) sums[wave * KO * 32 + k * 32 + q * 8 + e] = s;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < p.out; c += 256)
      p.db[(int64_t)blockIdx.x * p.out + c] = sums[c] + sums[KO * 32 + c] + sums[2 * KO * 32 + c] + sums[3 * KO * 32 + c];
  }
}

// f with the 32s of features in and out as constants.
template <typename F>
void with_widths(int in, int out, F f) {
  const int ki = (in + 31) / 32, ko = (out + 31) / 32;
  auto second = [&](auto k) {
    if (ko == 1) f(k, Number<1>());
    else if (ko == 2) f(k, Number<2>());
    else if (ko == 3) f(k, Number<3>());
    else f(k, Number<4>());
  };
  if (ki == 1) second(Number<1>());
  else if (ki == 2) second(Number<2>());
  else if (ki == 3) second(Number<3>());
  else second(Number<4>());
}

template <typename T>
hipError_t launch_narrow_layer(const LinearParams& p, hipStream_t s) {
  NarrowLayer<T> n{};
  n.x = static_cast<const T*>(p.x);
  n.w = static_cast<const T*>(p.w);
  n.rows = p.rows;
  n.in = p.in;
  n.out = p.out;
  n.act = p.activation;
  n.bias = static_cast<const T*>(p.bias);
  n.residual = static_cast<const T*>(p.residual);
  n.y = static_cast<T*>(p.y);
  n.kept = p.slope_bytes ? static_cast<uint8_t*>(p.kept) : nullptr;
  with_widths(p.in, p.out, [&](auto ki, auto ko) {
    constexpr int kRows = 64 * forward_groups(ki.value, ko.value);
    const int64_t turns = (p.rows + kRows - 1) / kRows;
    // Workgroups a CU: three with slopes to keep, else four.  us of both: kept,
    // 640,000 x 32 -> 128 69 and 75, 1,702,400 x 64 119 and 130; not kept,
    // 640,000 x 32 -> 128 63 and 60, x 128 -> 128 88 and 86, 1,702,400 x 64 99 and 100.
    const int64_t most = 256 * (n.kept ? 3 : 4);
    const unsigned grid = (unsigned)(turns < most ? turns : most);
    if (n.kept) narrow_layer_kernel<T, ki.value, ko.value, true><<<grid, 256, 0, s>>>(n);
    else narrow_layer_kernel<T, ki.value, ko.value, false><<<grid, 256, 0, s>>>(n);
  });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_narrow_layer_backward(const LinearParams& p, const LinearLayout& l, hipStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  NarrowLayer<T> n{};
  n.x = static_cast<const T*>(p.x);
  n.w = static_cast<const T*>(p.w);
  n.bias = static_cast<const T*>(p.bias);
  n.codes = p.codes;
  n.steps = p.steps;
  n.rows = p.rows;
  n.in = p.in;
  n.out = p.out;
  n.act = p.activation;
  n.dy = static_cast<const T*>(p.dy);
  n.slopes = static_cast<const uint8_t*>(p.kept);
  n.dx = static_cast<T*>(p.dx);
  n.dw = p.dw ? reinterpret_cast<float*>(ws + l.part) : nullptr;
  n.db = p.db ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
  with_widths(p.in, p.out, [&](auto ki, auto ko) {
    if (p.slope_bytes || p.codes) narrow_layer_backward_kernel<T, ki.value, ko.value, true><<<l.sum_rows, 256, 0, s>>>(n);
    else narrow_layer_backward_kernel<T, ki.value, ko.value, false><<<l.sum_rows, 256, 0, s>>>(n);
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  SumTasks t{};
  int k = 0;
  if (p.dw) t.t[k++] = {n.dw, l.sum_rows, 1, p.in * p.out, nullptr, nullptr, p.dw, nullptr};
  if (p.db) t.t[k++] = {n.db, l.sum_rows, 1, p.out, nullptr, nullptr, p.db, nullptr};
  return k ? launch_column_sums<T>(t, k, s) : hipSuccess;
}

}  // namespace
}  // namespace nest
