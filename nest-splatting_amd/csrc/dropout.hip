// Dropout from a counter-based generator, with an optional residual:
//
//   y[i] = keep(i) ? x[i] * scale : 0   (+ residual[i])
//
// keep(i) compares a 16-bit random number with a threshold t = round(65536 p);
// scale = 65536 / (65536 - t), so the mean is kept exactly for the share that
// is kept in fact.  Elements 8 c to 8 c + 7 take the eight halves of one
// 128-bit block of Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) at the counter
// (c, offset) under the key seed.  Nothing about the mask is stored: the
// backward pass is the same kernel on dy with the same seed and offset.
//
// A thread makes one block and moves its eight elements in 16-byte vectors.
// A dropped element is selected away, not multiplied by zero, so an infinity
// or NaN there does not reach the output.  The sum with the residual is
// rounded once.
//
// Bound by memory: 1,702,400 x 64 bf16 with a residual 114 us (5.8 TB/s of
// x, residual and y), its backward 73 us (5.9 TB/s); the generator's twenty
// 64-bit products per eight elements hide behind the loads.  Thirty-two bits an
// element would need two blocks for a 16-byte vector of a 16-bit type.
#include "blocks_internal.h"
#include "vec_io.h"

namespace nest {
namespace {

constexpr int64_t kGrid = 1 << 22;

__device__ __forceinline__ void philox4x32(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    c[0] = (uint32_t)(p1 >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)p1;
    c[2] = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

template <typename T, bool kResidual>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutParams p) {
  constexpr int N = Vec16<T>::kN, kV = 8 / N;
  // The grid covers all blocks up to kGrid workgroups; past that it strides.
  for (int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x; block * 8 < p.n; block += (int64_t)gridDim.x * 256) {
  const int64_t at = block * 8;
  const int left = p.n - at < 8 ? (int)(p.n - at) : 8;
  const T* x = static_cast<const T*>(p.x) + at;
  const T* res = static_cast<const T*>(p.residual) + at;
  T* y = static_cast<T*>(p.y) + at;
  float v[kV][N], r[kV][N];
#pragma unroll
  for (int k = 0; k < kV; k++) {
    load_vec<T>(v[k], x + k * N, left - k * N);
    if constexpr (kResidual) load_vec<T>(r[k], res + k * N, left - k * N);
  }
  uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), (uint32_t)p.offset, (uint32_t)(p.offset >> 32)};
  philox4x32(c, (uint32_t)p.seed, (uint32_t)(p.seed >> 32));
#pragma unroll
  for (int k = 0; k < kV; k++) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int e = k * N + i;
      const uint32_t u = (e & 1) ? c[e >> 1] >> 16 : c[e >> 1] & 0xffffu;
      const float d = u >= p.threshold ? v[k][i] * p.scale : 0.0f;
      v[k][i] = kResidual ? r[k][i] + d : d;
    }
    store_vec<T>(y + k * N, v[k], left - k * N);
  }
  }
}

template <typename T>
hipError_t launch(const DropoutParams& p, hipStream_t s) {
  const int64_t need = (p.n + 2047) / 2048;
  const unsigned grid = (unsigned)(need < kGrid ? need : kGrid);
  if (p.residual) dropout_kernel<T, true><<<grid, 256, 0, s>>>(p);
  else dropout_kernel<T, false><<<grid, 256, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const DropoutParams& p, hipStream_t s) {
  if (p.dtype == NEST_DTYPE_F32) return launch<float>(p, s);
  return p.dtype == NEST_DTYPE_F16 ? launch<f16_t>(p, s) : launch<bf16_t>(p, s);
}

}  // namespace nest
