// The dense layer for narrow rows (at most 64 features in and out) of float32:
// rows stay in registers, weights in LDS, as in linear_narrow.h.
//
// The products run on the float32 matrix instruction of 16 x 16 x 4, an eighth
// of the bf16 rate but without the three parts a value of the tiles: rows of
// this width are bound by memory all the same.  A lane's four floats of a row
// are the operands of four instructions, whatever order that gives the sum
// over features, since the weights come in the same order; and a lane's
// accumulators of a product are four consecutive features of its row, the
// layout that it loads, stores and hands to the next product.  The weights'
// gradient sums over rows: a wave puts its 16 rows of dz and x into LDS of its
// own and reads them by columns, so no barrier stands in the loop; the waves'
// sums are joined at the end, in their order.
//
// us of a forward and a backward here and in tiles, GELU: 640,000 x 64 -> 64 127 +
// 149 and 132 + 259, 32 -> 32 48 + 67 and 73 + 170, 16 -> 64 93 + 85 and 114 +
// 231, 16 rows of 64 -> 64 13 + 19 and 14 + 27.  Memory bound past the exact
// GELU (with ReLU 95 us: 369 MB at 3.9 TB/s).
//
// Slopes are kept and read as in the tiles.  (Made again from x they would save
// a third of a backward's bytes; the tiles' callers keep float32 slopes at any
// width.)
#pragma once

#include "linear_narrow.h"

namespace nest {
namespace {

struct NarrowF32 {
  const float *x, *w;        // a backward's x may be null: codes hold it, or nothing asks for it
  const int8_t* codes;
  const uint8_t* steps;
  int64_t rows;
  int in, out;
  Epilogue<float> ep;        // forward
  const float* dy;           // backward
  const void* slopes;        // or null: none
  int slope_bytes;
  float* dx;
  float *dw, *db;            // [groups][out][in], [groups][out]; each may be null
};

// A [rows][cols] matrix of the weights (transposed: [cols][rows] in memory) to
// LDS, zeros around it; pitches of an odd number of 16 bytes.
template <int R, int C, bool kTransposed>
__device__ __forceinline__ void stage_weights_f32(float* lds, const float* w, int rows, int cols) {
  constexpr int kPitch = C + 4, kLong = kTransposed ? R : C, kPieces = (R * C + 4 * 256 - 1) / (4 * 256);
  const int length = kTransposed ? rows : cols, lines = kTransposed ? cols : rows;
  Words16<float> v[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; u++) {
    const int i = (u * 256 + threadIdx.x) * 4, line = i / kLong, at = i % kLong;
    v[u] = load_words<false>(w + line * length + at, line < lines ? length - at : 0);
  }
#pragma unroll
  for (int u = 0; u < kPieces; u++) {
    const int i = (u * 256 + threadIdx.x) * 4, line = i / kLong, at = i % kLong;
    if (i >= R * C) break;
    if constexpr (kTransposed) {
#pragma unroll
      for (int e = 0; e < 4; e++) lds[(at + e) * kPitch + line] = v[u][e];
    } else {
      *reinterpret_cast<f32x4*>(lds + line * kPitch + at) = __builtin_bit_cast(f32x4, v[u]);
    }
  }
}

// 4 bytes of a row with n left at p, zeros past its end.
__device__ __forceinline__ uint32_t row_word(const void* p, int n) {
  uint32_t v = 0;
  if (n >= 4) {
    __builtin_memcpy(&v, p, 4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) v |= (uint32_t)static_cast<const uint8_t*>(p)[i] << (i * 8);
  }
  return v;
}

// Features 16 J + 4 (lane / 16) + 0..3 of row lane % 16, over K features.
template <int K>
__device__ __forceinline__ f32x4 narrow_product_f32(const float* lds, int J, const f32x4 (&row)[K / 16]) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < K / 16; k++) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(lds + (16 * J + r) * (K + 4) + k * 16 + q * 4);
#pragma unroll
    for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], row[k][e], acc, 0, 0, 0);
  }
  return acc;
}

// Results pass through LDS of the wave's own, so that a lane has 16 bytes of a
// row and the lanes a row's in a line: 64 of each of 16 rows took 162 us for
// 640,000 x 64 -> 64 with GELU, where so it takes 127.
template <int KI, int KO>
__global__ __launch_bounds__(256, 4) void narrow_f32_kernel(NarrowF32 p) {
  constexpr int kPitch = KO * 16 + 4, kRow = KO * 4;   // pieces of 4 floats
  __shared__ __attribute__((aligned(16))) float w[KO * 16 * (KI * 16 + 4)], stages[4][16 * kPitch];
  stage_weights_f32<KO * 16, KI * 16, false>(w, p.w, p.out, p.in);
  __syncthreads();
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int64_t step = (int64_t)gridDim.x * 64;
  Words16<float> next[KI];
  auto load = [&](int64_t at) {
#pragma unroll
    for (int k = 0; k < KI; k++) next[k] = load_words<false>(p.x + at * p.in + k * 16 + q * 4, at < p.rows ? p.in - k * 16 - q * 4 : 0);
  };
  int64_t row = ((int64_t)blockIdx.x * 4 + wave_id()) * 16 + r;
  load(row);
  for (; row - r < p.rows; row += step) {
    f32x4 x[KI];
#pragma unroll
    for (int k = 0; k < KI; k++) x[k] = __builtin_bit_cast(f32x4, next[k]);
    load(row + step);   // on its way while these rows are worked on
    float* const stage = stages[wave_id()];
#pragma unroll
    for (int J = 0; J < KO; J++) *reinterpret_cast<f32x4*>(&stage[r * kPitch + J * 16 + q * 4]) = narrow_product_f32<KI * 16>(w, J, x);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    with_activation(p.ep.act, [&](auto act) {
#pragma unroll
      for (int u = 0; u < KO; u++) {
        const int t = u * 64 + lane, at = t / kRow, c = t % kRow * 4;
        const f32x4 v = *reinterpret_cast<const f32x4*>(&stage[at * kPitch + c]);
        float z[4] = {v[0], v[1], v[2], v[3]};
        if (row - r + at < p.rows && c < p.out) p.ep.template finish<4, act.value>(row - r + at, c, p.out - c, z);
      }
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// A tile's pitch: four rows of 16 floats one after another fall on different banks.
constexpr int f32_pitch(int cols) { return cols % 32 ? cols : cols + 16; }

template <int KI, int KO>
__global__ __launch_bounds__(256, narrow_f32_groups(KI, KO)) void narrow_f32_backward_kernel(NarrowF32 p) {
  constexpr int PO = f32_pitch(KO * 16), PI = f32_pitch(KI * 16);
  __shared__ __attribute__((aligned(16))) float wt[KI * 16 * (KO * 16 + 4)];
  __shared__ __attribute__((aligned(16))) float tz[4][16 * PO], tx[4][16 * PI];   // a wave's rows
  __shared__ float sums[KO * KI * 256];
  if (p.dx) stage_weights_f32<KI * 16, KO * 16, true>(wt, p.w, p.in, p.out);
  __syncthreads();
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = wave_id();
  const int64_t step = (int64_t)gridDim.x * 64;
  const int groups_in = (p.in + 31) / 32;
  Words16<float> nx[KI], ndy[KO], ns[KO];   // of fewer bytes a value: the first of the words
  int nstep[KI];
  auto load = [&](int64_t at) {
    const bool in = at < p.rows;
    auto left = [&](int k, int cols) { return in ? cols - k * 16 - q * 4 : 0; };
    auto place = [&](int k, int cols) { return at * cols + k * 16 + q * 4; };
#pragma unroll
    for (int k = 0; k < KO; k++) ndy[k] = load_words<false>(p.dy + place(k, p.out), left(k, p.out));
    if (p.codes) {
#pragma unroll
      for (int k = 0; k < KI; k++) {
        nx[k].w[0] = row_word(p.codes + place(k, p.in), left(k, p.in));
        nstep[k] = left(k, p.in) > 0 ? p.steps[at * groups_in + k / 2] : 0;
      }
    } else {
#pragma unroll
      for (int k = 0; k < KI; k++) nx[k] = load_words<false>(p.x + place(k, p.in), p.x ? left(k, p.in) : 0);
    }
    if (p.slope_bytes == 4) {
#pragma unroll
      for (int k = 0; k < KO; k++) ns[k] = load_words<false>(static_cast<const float*>(p.slopes) + place(k, p.out), left(k, p.out));
    } else if (p.slope_bytes == 2) {
#pragma unroll
      for (int k = 0; k < KO; k++) {
        const uint2 v = row_bytes(static_cast<const int16_t*>(p.slopes) + place(k, p.out), left(k, p.out) * 2);
        ns[k].w[0] = v.x;
        ns[k].w[1] = v.y;
      }
    } else if (p.slope_bytes == 1) {
#pragma unroll
      for (int k = 0; k < KO; k++) ns[k].w[0] = row_word(static_cast<const uint8_t*>(p.slopes) + place(k, p.out), left(k, p.out));
    }
  };
  f32x4 dw[KO][KI] = {};
  float db[KO][4] = {};
  int64_t row = ((int64_t)blockIdx.x * 4 + wave) * 16 + r;
  load(row);
  for (; row - r < p.rows; row += step) {
    f32x4 x[KI], dz[KO];
#pragma unroll
    for (int k = 0; k < KI; k++) {
      x[k] = __builtin_bit_cast(f32x4, nx[k]);
      if (p.codes) {
        const float unit = nstep[k] == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.0f, nstep[k] - 132);
#pragma unroll
        for (int e = 0; e < 4; e++) x[k][e] = (float)(int8_t)(nx[k].w[0] >> (e * 8)) * unit;   // past the row's end of no gradient that is stored
      }
    }
    auto make_dz = [&](auto slope) {
#pragma unroll
      for (int k = 0; k < KO; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          dz[k][e] = ndy[k][e] * slope(k, e);   // zero past the ends
          db[k][e] += dz[k][e];
        }
    };
    if (p.slope_bytes == 4) make_dz([&](int k, int e) { return ns[k][e]; });
    else if (p.slope_bytes == 2) make_dz([&](int k, int e) { return slope_of((int16_t)(ns[k].w[e / 2] >> (e % 2 * 16))); });
    else if (p.slope_bytes == 1) make_dz([&](int k, int e) { return coarse_slope((float)((ns[k].w[0] >> (e * 8)) & 0xffu)); });
    else make_dz([&](int, int) { return 1.0f; });
    if (p.dw) {
#pragma unroll
      for (int k = 0; k < KO; k++) *reinterpret_cast<f32x4*>(&tz[wave][r * PO + k * 16 + q * 4]) = dz[k];
#pragma unroll
      for (int k = 0; k < KI; k++) *reinterpret_cast<f32x4*>(&tx[wave][r * PI + k * 16 + q * 4]) = x[k];
    }
    load(row + step);   // on its way while these rows are worked on
    if (p.dx) {
#pragma unroll
      for (int J = 0; J < KI; J++) {
        const f32x4 acc = narrow_product_f32<KO * 16>(wt, J, dz);
        const int c = J * 16 + q * 4;
        const float v[4] = {acc[0], acc[1], acc[2], acc[3]};
        store_vec<float>(p.dx + row * p.in + c, v, row < p.rows ? p.in - c : 0);
      }
    }
    if (p.dw) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < 4; t++) {   // rows 4 t + lane / 16
        float a[KO], b[KI];
#pragma unroll
        for (int i = 0; i < KO; i++) a[i] = tz[wave][(t * 4 + q) * PO + i * 16 + r];
#pragma unroll
        for (int j = 0; j < KI; j++) b[j] = tx[wave][(t * 4 + q) * PI + j * 16 + r];
#pragma unroll
        for (int i = 0; i < KO; i++)
#pragma unroll
          for (int j = 0; j < KI; j++) dw[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[i], dw[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // dw[i][j]: output feature 16 i + lane % 16, input features 16 j + 4 (lane / 16) + 0..3
  if (p.dw) {
    for (int v = 0; v < 4; v++) {
      if (wave == v) {
#pragma unroll
        for (int i = 0; i < KO; i++)
#pragma unroll
          for (int j = 0; j < KI; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float* const at = &sums[((i * KI + j) * 4 + e) * 64 + lane];
              *at = v ? *at + dw[i][j][e] : dw[i][j][e];
            }
      }
      __syncthreads();
    }
    float* const part = p.dw + (int64_t)blockIdx.x * p.out * p.in;
    for (int t = threadIdx.x; t < KO * KI * 256; t += 256) {
      const int l = t & 63, e = t >> 6 & 3, tile = t >> 8, o = tile / KI * 16 + (l & 15), c = tile % KI * 16 + (l >> 4) * 4 + e;
      if (o < p.out && c < p.in) part[o * p.in + c] = sums[t];
    }
    __syncthreads();
  }
  if (p.db) {
#pragma unroll
    for (int k = 0; k < KO; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float s = db[k][e];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
        if (r == 0) sums[wave * KO * 16 + k * 16 + q * 4 + e] = s;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < p.out; c += 256)
      p.db[(int64_t)blockIdx.x * p.out + c] = sums[c] + sums[KO * 16 + c] + sums[2 * KO * 16 + c] + sums[3 * KO * 16 + c];
  }
}

// f with the 16s of features in and out as constants.
template <typename F>
void with_widths_f32(int in, int out, F f) {
  const int ki = (in + 15) / 16, ko = (out + 15) / 16;
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

// Templates, so that a unit of another type makes none of these kernels.
template <typename T>
hipError_t launch_narrow_f32(const LinearParams& p, const Epilogue<T>& ep, hipStream_t s) {
  static_assert(sizeof(T) == 4, "");
  NarrowF32 n{};
  n.x = static_cast<const float*>(p.x);
  n.w = static_cast<const float*>(p.w);
  n.rows = p.rows;
  n.in = p.in;
  n.out = p.out;
  n.ep = ep;
  const int64_t turns = (p.rows + 63) / 64;
  const unsigned grid = (unsigned)(turns < 256 * 8 ? turns : 256 * 8);   // 640,000 x 16 -> 64 95 us, with four a CU 107
  with_widths_f32(p.in, p.out, [&](auto ki, auto ko) { narrow_f32_kernel<ki.value, ko.value><<<grid, 256, 0, s>>>(n); });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_narrow_f32_backward(const LinearParams& p, const LinearLayout& l, hipStream_t s) {
  static_assert(sizeof(T) == 4, "");
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  NarrowF32 n{};
  n.x = p.dw ? static_cast<const float*>(p.x) : nullptr;
  n.w = static_cast<const float*>(p.w);
  n.codes = p.dw ? p.codes : nullptr;
  n.steps = p.steps;
  n.rows = p.rows;
  n.in = p.in;
  n.out = p.out;
  n.dy = static_cast<const float*>(p.dy);
  n.slopes = p.kept;
  n.slope_bytes = p.slope_bytes;
  n.dx = static_cast<float*>(p.dx);
  n.dw = p.dw ? reinterpret_cast<float*>(ws + l.part) : nullptr;
  n.db = p.db ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
  with_widths_f32(p.in, p.out, [&](auto ki, auto ko) { narrow_f32_backward_kernel<ki.value, ko.value><<<l.sum_rows, 256, 0, s>>>(n); });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  SumTasks t{};
  int k = 0;
  if (p.dw) t.t[k++] = {n.dw, l.sum_rows, 1, p.in * p.out, nullptr, nullptr, p.dw, nullptr};
  if (p.db) t.t[k++] = {n.db, l.sum_rows, 1, p.out, nullptr, nullptr, p.db, nullptr};
  return k ? launch_column_sums<float>(t, k, s) : hipSuccess;
}

}  // namespace
}  // namespace nest
