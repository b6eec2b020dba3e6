// Sums of partial rows by column, for the gradients of what rows share
// (residual_norm.hip, linear_calls.h).
#pragma once

#include "vec_io.h"

namespace nest {
namespace {

// For each of `groups` groups the sum of n rows, each times its row of
// `weight` where there is one: out0 = the sum times mul0 and out1 times mul1
// by column, and the sum itself.
struct SumTask {
  const float* part;
  int64_t n, groups;
  int cols;
  const void *weight, *mul0, *mul1;
  void *out0, *out1;
  float* sum;
};
struct SumTasks {
  SumTask t[2];
};

// 32 columns a workgroup, 32 slices of the rows, joined in LDS in their order.
template <typename P>
__global__ __launch_bounds__(1024) void column_sums_kernel(SumTasks tasks) {
  __shared__ float lds[32][33];
  const SumTask& t = tasks.t[blockIdx.z];
  const int64_t D = t.cols;
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  for (int64_t g = blockIdx.y; g < t.groups; g += gridDim.y) {
    const float* part = t.part + g * t.n * D + col;
    float s = 0.0f;
    if (col < D) {
      int64_t r = slice;
      if (!t.weight)
        for (; r + 7 * 32 < t.n; r += 8 * 32) {   // eight loads in flight
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] = part[(r + i * 32) * D];
#pragma unroll
          for (int i = 0; i < 8; i++) s += v[i];
        }
      for (; r < t.n; r += 32) {
        const float v = part[r * D];
        s = t.weight ? fmaf(v, to_f32(static_cast<const P*>(t.weight)[r * D + col]), s) : s + v;
      }
    }
    __syncthreads();   // the last group's sums are all read
    lds[slice][threadIdx.x & 31] = s;
    __syncthreads();
    if (slice == 0 && col < D) {
      float all = 0.0f;
#pragma unroll
      for (int r = 0; r < 32; r++) all += lds[r][threadIdx.x];
      auto out = [&](void* to, const void* mul) {
        if (to) static_cast<P*>(to)[g * D + col] = from_f32<P>(mul ? all * to_f32(static_cast<const P*>(mul)[col]) : all);
      };
      out(t.out0, t.mul0);
      out(t.out1, t.mul1);
      if (t.sum) t.sum[g * D + col] = all;
    }
  }
}

template <typename P>
hipError_t launch_column_sums(const SumTasks& tasks, int n, hipStream_t s) {
  int64_t groups = 1;
  int cols = 1;
  for (int i = 0; i < n; i++) {
    groups = tasks.t[i].groups > groups ? tasks.t[i].groups : groups;
    cols = tasks.t[i].cols > cols ? tasks.t[i].cols : cols;
  }
  column_sums_kernel<P><<<dim3((unsigned)((cols + 31) / 32), (unsigned)(groups < 4096 ? groups : 4096), n), 1024, 0, s>>>(tasks);
  return hipGetLastError();
}

}  // namespace
}  // namespace nest
