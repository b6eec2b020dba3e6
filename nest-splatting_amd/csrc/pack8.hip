// Rows held in 8 bits, and back.
//
// 32 consecutive values of a row share a step, the power of two 2^(e - 6) with
// e = floor(log2 of the largest magnitude) (-126 at least); a value is held as
// the nearest whole number of steps, halves to the even one, -127 to 127, so
// the largest takes 64 to 127 of them.  A value is off by at most half a step,
// 2^-7 of its group's largest; one within 2^-8 of the next power of two is off
// by at most a whole step, where its 128 steps do not fit.  A power of two
// makes both scalings exact: what comes back is a function of x alone, in
// either 16-bit type too, which hold all 7 bits of it.  The step is held as
// e + 126; 255 stands for a group with an infinity or a NaN, which comes back
// as NaN.
//
// Memory bound: 16 values a lane, one 16-byte piece of codes.  1,702,400 x 64 of
// bf16: 71 us there (330 MB: 4.7 TB/s) and 62 back (5.3 TB/s).
#include "residual_internal.h"
#include "vec_io.h"

namespace nest {
namespace {

constexpr int kThreads = 256, kValues = 16, kHalves = kPackGroup / kValues;
constexpr uint32_t kNotFinite = 255;

struct alignas(1) Codes {
  int8_t v[kValues];
};

// 16 values of a row with n left at p, the rest zero.
template <typename T>
__device__ __forceinline__ void load16(float (&f)[kValues], const T* p, int n) {
  constexpr int N = Vec16<T>::kN;
#pragma unroll
  for (int k = 0; k < kValues / N; k++) {
    const Words16<T> t = load_words<false>(p + k * N, n - k * N);
#pragma unroll
    for (int i = 0; i < N; i++) f[k * N + i] = to_f32(t[i]);
  }
}

// Row and first column of a half group; `halves` to a row.
struct Place {
  int64_t row;
  int col;
};
__device__ __forceinline__ Place place_of(int64_t i, uint32_t halves, bool small) {
  const int64_t row = small ? (int64_t)((uint32_t)i / halves) : i / halves;
  return {row, (int)(i - row * halves) * kValues};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack8_kernel(int64_t rows, int cols, const T* x, int8_t* codes, uint8_t* steps) {
  const uint32_t halves = (uint32_t)((cols + kPackGroup - 1) / kPackGroup) * kHalves;
  const int64_t total = rows * halves;   // even, so both lanes of a group take part
  const bool small = total < (int64_t)1 << 32;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const Place at = place_of(i, halves, small);
    const int left = cols - at.col;
    float v[kValues];
    load16(v, x + at.row * cols + at.col, left);
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kValues; k++) {
      const uint32_t m = __builtin_bit_cast(uint32_t, v[k]) & 0x7fffffffu;
      most = m > most ? m : most;
    }
    const uint32_t other = (uint32_t)__shfl_xor((int)most, 1);
    most = other > most ? other : most;
    uint32_t step = most >> 23;
    step = step == kNotFinite ? kNotFinite : (step > 1 ? step - 1 : 0);   // e + 126
    Codes c;
#pragma unroll
    for (int k = 0; k < kValues; k++) {
      const float q = __builtin_rintf(__builtin_amdgcn_ldexpf(v[k], 132 - (int)step));
      c.v[k] = step == kNotFinite ? (int8_t)0 : (int8_t)__builtin_amdgcn_fmed3f(q, -127.0f, 127.0f);
    }
    int8_t* to = codes + at.row * cols + at.col;
    if (left >= kValues) {
      store_whole(to, c);
    } else {
#pragma unroll
      for (int k = 0; k < kValues; k++)
        if (k < left) to[k] = c.v[k];
    }
    if ((i & 1) == 0) steps[i >> 1] = (uint8_t)step;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(int64_t rows, int cols, const int8_t* codes, const uint8_t* steps, T* y,
                                                           int64_t ldy) {
  constexpr int N = Vec16<T>::kN;
  const uint32_t halves = (uint32_t)((cols + kPackGroup - 1) / kPackGroup) * kHalves;
  const int64_t total = rows * halves;
  const bool small = total < (int64_t)1 << 32;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const Place at = place_of(i, halves, small);
    const int left = cols - at.col;
    const int8_t* from = codes + at.row * cols + at.col;
    Codes c;
    if (left >= kValues) {
      __builtin_memcpy(&c, from, kValues);
    } else {
#pragma unroll
      for (int k = 0; k < kValues; k++) c.v[k] = k < left ? from[k] : (int8_t)0;
    }
    const uint32_t step = steps[i >> 1];
    T* to = y + at.row * ldy + at.col;
    const int n = (int)(ldy - at.col);   // the row's end and its zeros
#pragma unroll
    for (int k = 0; k < kValues / N; k++) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float v = __builtin_amdgcn_ldexpf((float)c.v[k * N + j], (int)step - 132);
        f[j] = step == kNotFinite && k * N + j < left ? __builtin_nanf("") : v;
      }
      store_vec<T>(to + k * N, f, n - k * N);
    }
  }
}

unsigned grid_of(int64_t rows, int cols) {
  const int64_t need = (rows * pack_groups(cols) * kHalves + kThreads - 1) / kThreads;
  return (unsigned)(need < 16384 ? need : 16384);
}

}  // namespace

hipError_t launch_pack8(int64_t rows, int cols, int dtype, const void* x, int8_t* codes, uint8_t* steps, hipStream_t s) {
  const unsigned grid = grid_of(rows, cols);
  if (dtype == NEST_DTYPE_F32) pack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, static_cast<const float*>(x), codes, steps);
  else if (dtype == NEST_DTYPE_F16) pack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, static_cast<const f16_t*>(x), codes, steps);
  else pack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, static_cast<const bf16_t*>(x), codes, steps);
  return hipGetLastError();
}

hipError_t launch_unpack8(int64_t rows, int cols, int dtype, const int8_t* codes, const uint8_t* steps, void* y, int64_t ldy,
                          hipStream_t s) {
  const unsigned grid = grid_of(rows, cols);
  if (dtype == NEST_DTYPE_F32) unpack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, codes, steps, static_cast<float*>(y), ldy);
  else if (dtype == NEST_DTYPE_F16) unpack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, codes, steps, static_cast<f16_t*>(y), ldy);
  else unpack8_kernel<<<grid, kThreads, 0, s>>>(rows, cols, codes, steps, static_cast<bf16_t*>(y), ldy);
  return hipGetLastError();
}

}  // namespace nest
