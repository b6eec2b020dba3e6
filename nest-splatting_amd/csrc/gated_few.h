// The gated feed-forward block for few rows (a token, a small batch): bound by
// reading the weights once.
//
// The weights go straight from memory to registers, as no value is used twice;
// on MFMA, with the weights as the first operand and the rows of x as the
// second, the products cost nothing beside the loads.  The 16 first-operand
// rows of an instruction are 16 / S weight rows in S parts of k each, and so
// are the 16 columns: the diagonal blocks of the result, where both parts
// agree, are summed, the rest is of no use.  With S = 16 (one row of x) a load
// takes 1 KB of one weight row, with S = 4 (up to four) 256 bytes of four, with
// S = 2 (up to 16) 128 bytes of eight.  S = 1, 64 bytes of sixteen rows, would
// fit 16 rows of x, but a line's halves then come by two loads between which
// the L1 may lose it: 38 us instead of 29 for 16 rows of 2048 -> 8192 bf16.
// Waves of a workgroup share k and join their sums in LDS in their order.  One
// launch for the gate, one for the down projection.
//
// Measured, 2048 -> 8192: one row bf16 13.3 us for the gate (67 MB, 5.0 TB/s)
// and 9.6 for the down projection (33 MB).
#pragma once

#include "gated_tiles.h"

namespace nest {
namespace {

template <typename T>
struct Few {
  const T* x;             // [M][ldx] activations (x, or h with its zero padding)
  const T *w0, *w1;       // [N][K]: Wg and Wu, or Wd and null
  int64_t ldx;
  int M, N, K;
  T* out;                 // [M][ldo]: h or y
  int64_t ldo;
  float* kept;            // the gate's, see kept_block; or null
  int act;
};

// 16 bytes at p of a row with n values left.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag load_frag(const T* p, int n) {
  constexpr int kVec = 16 / (int)sizeof(T);
  typename Mma<T>::Frag f;
  if (n >= kVec) {
    __builtin_memcpy(&f, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i++) f[i] = i < n ? p[i] : (T)0.0f;
  }
  return f;
}

// Shapes: S parts, NB blocks of 16 / S rows of x, RT groups of 16 / S weight
// rows a wave, U loads of each in flight.
template <int kS, int kNB, int kRT, int kU>
struct FewShape {
  static constexpr int S = kS, NB = kNB, RT = kRT, U = kU, TR = 16 / kS, rows = TR * kRT, columns = TR * kNB;
};
constexpr int kFewWaves = 8;   // of a workgroup at most

template <typename T, typename C, bool kGate>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(Few<T> p) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int S = C::S, NB = C::NB, RT = C::RT, U = C::U, TR = C::TR;
  constexpr int kVec = 16 / (int)sizeof(T), kLoad = S * 4 * kVec, kChunk = kLoad * U, kMats = kGate ? 2 : 1;
  constexpr int kOut = C::rows * C::columns;
  __shared__ float sums[kFewWaves][kMats][kOut];
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, waves = blockDim.x >> 6, w = wave_id();
  const int sub = r / S, part = r % S;
  const int64_t n0 = (int64_t)blockIdx.x * C::rows;
  f32x4 acc[kMats][RT][NB] = {};
  for (int64_t chunk = (int64_t)w * kChunk; chunk < p.K; chunk += (int64_t)waves * kChunk) {
    const int64_t k0 = chunk + part * (4 * kVec) + q * kVec;
    Frag fw[kMats][RT][U], fx[NB][U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int64_t k = k0 + i * kLoad;
      const int left = k < p.K ? (int)(p.K - k) : 0;
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int m = 0; m < kMats; m++) {
          const int64_t n = n0 + t * TR + sub;
          fw[m][t][i] = load_frag<T>((m ? p.w1 : p.w0) + n * p.K + k, n < p.N ? left : 0);
        }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int64_t k = k0 + i * kLoad;
      const int left = k < p.K ? (int)(p.K - k) : 0;
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const int64_t n = b * TR + sub;
        fx[b][i] = load_frag<T>(p.x + n * p.ldx + k, n < p.M ? left : 0);
      }
    }
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int m = 0; m < kMats; m++)
#pragma unroll
          for (int b = 0; b < NB; b++) acc[m][t][b] = Mma<T>::run(fw[m][t][i], fx[b][i], acc[m][t][b]);
  }
  // the diagonal blocks: element e of a lane is first-operand row 4 q + e
#pragma unroll
  for (int m = 0; m < kMats; m++)
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const f32x4 v = acc[m][t][b];
        if constexpr (S == 2) {
          // weight rows 2 q and 2 q + 1, parts 0 and 1 of each
          float d0 = part ? v[1] : v[0], d1 = part ? v[3] : v[2];
          d0 += __shfl_xor(d0, 1);
          d1 += __shfl_xor(d1, 1);
          if (part == 0) {
            sums[w][m][(t * TR + q * 2) * C::columns + b * TR + sub] = d0;
            sums[w][m][(t * TR + q * 2 + 1) * C::columns + b * TR + sub] = d1;
          }
        } else {
          static_assert(S == 4 || S == 16, "");
          // weight row q * 4 / S, parts 4 q % S + e
          float d = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e++) d = (q * 4 + e) % S == part ? v[e] : d;
          for (int o = 1; o < S; o <<= 1) d += __shfl_xor(d, o);
          if constexpr (S == 16) {
            d += __shfl_xor(d, 16);
            d += __shfl_xor(d, 32);
          }
          if (part == 0 && (S == 4 || q == 0)) sums[w][m][(t * TR + (S == 4 ? q : 0)) * C::columns + b * TR + sub] = d;
        }
      }
  __syncthreads();
  with_act(p.act, [&](auto act) {
    for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
      const int64_t c = n0 + o / C::columns;
      const int row = o % C::columns;
      float v[kMats] = {};
      for (int i = 0; i < waves; i++)
#pragma unroll
        for (int m = 0; m < kMats; m++) v[m] += sums[i][m][o];
      if constexpr (kGate) {
        if (c >= p.ldo) continue;
        if (p.kept) {
          const int64_t at = ((row >> 4) * ((p.ldo + 15) >> 4) + (c >> 4)) * 512 + (((c & 15) >> 2) * 16 + (row & 15)) * 4 + (c & 3);
          p.kept[at] = v[0];
          p.kept[at + 256] = v[1];
        }
        float unused;
        v[0] = c < p.N ? act_value<T, act.value, false>(v[0], unused) * v[1] : 0.0f;
        if (row < p.M) p.out[row * p.ldo + c] = from_f32<T>(v[0]);
      } else if (row < p.M && c < p.N) {
        p.out[row * p.ldo + c] = from_f32<T>(v[0]);
      }
    }
  });
}

template <typename T, typename C, bool kGate>
hipError_t launch_few_shape(const Few<T>& p, hipStream_t s) {
  constexpr int kChunk = 64 / (int)sizeof(T) * C::S * C::U;
  const int64_t tiles = ((kGate ? p.ldo : p.N) + C::rows - 1) / C::rows;
  int waves = 1;
  while (waves < kFewWaves && waves * kChunk < p.K) waves *= 2;
  few_kernel<T, C, kGate><<<(unsigned)tiles, waves * 64, 0, s>>>(p);
  return hipGetLastError();
}

template <typename T, bool kGate>
hipError_t launch_few(const Few<T>& p, hipStream_t s) {
  constexpr int kMore = kGate ? 1 : 2;
  if (p.M == 1) return launch_few_shape<T, FewShape<16, 1, 2 * kMore, 4>, kGate>(p, s);
  if (p.M <= 4) return launch_few_shape<T, FewShape<4, 1, 2 * kMore, 4>, kGate>(p, s);
  if (p.M <= 8) return launch_few_shape<T, FewShape<2, 1, 1, 8>, kGate>(p, s);
  return launch_few_shape<T, FewShape<2, 2, 1, 4>, kGate>(p, s);
}

template <typename T>
hipError_t launch_few_forward(const GatedParams& g, const GatedLayout& l, hipStream_t s) {
  T* h = reinterpret_cast<T*>(static_cast<uint8_t*>(g.ws) + l.h);
  const Few<T> gate{static_cast<const T*>(g.x), static_cast<const T*>(g.w_gate), static_cast<const T*>(g.w_up), g.in,
                    (int)g.rows, g.hidden, g.in, h, l.ldh, g.kept, g.activation};
  if (hipError_t e = launch_few<T, true>(gate, s); e != hipSuccess) return e;
  const Few<T> down{h, static_cast<const T*>(g.w_down), nullptr, l.ldh, (int)g.rows, g.out, g.hidden, static_cast<T*>(g.y), g.out,
                    nullptr, 0};
  return launch_few<T, false>(down, s);
}

}  // namespace
}  // namespace nest
