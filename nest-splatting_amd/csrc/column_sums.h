// Sums of partial rows by column, for the gradients of what rows share
// (residual_norm.hip, linear_calls.h).
#pragma once

#include "vec_io.h"

namespace nest {
namespace {

// For each of `groups` groups the sum of n rows (below 2^32), `shared` after
// another times one row of `weight` where there is one: out0 = the sum times mul0 and out1
// times mul1 by column.
struct SumTask {
  const float* part;
  int64_t n, groups;
  int cols;
  const void *weight, *mul0, *mul1;
  void *out0, *out1;
  uint32_t shared;
};
// Of a task; a workgroup takes every 4096th. 3 tasks of 256 workgroups across
// stay under 2^32 threads a launch.
constexpr int64_t kGroupsAtOnce = 4096;
struct SumTasks {
  SumTask t[3];
  unsigned first[3];   // workgroup of each task
};

template <typename P>
__device__ __forceinline__ float weight_of(const SumTask& t, uint32_t row, int64_t D, int col) {
  return to_f32(static_cast<const P*>(t.weight)[row / t.shared * D + col]);
}

// 32 columns a workgroup, 32 slices of the rows, joined in LDS in their order.
template <typename P>
__global__ __launch_bounds__(1024) void column_sums_kernel(SumTasks tasks) {
  __shared__ float lds[32][33];
  const int which = blockIdx.x >= tasks.first[2] ? 2 : blockIdx.x >= tasks.first[1] ? 1 : 0;
  const SumTask& t = tasks.t[which];
  const int64_t D = t.cols;
  const unsigned across = (unsigned)((D + 31) / 32), id = blockIdx.x - tasks.first[which];
  const int col = (int)(id % across) * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  const uint32_t n = (uint32_t)t.n;
  for (int64_t g = id / across; g < t.groups; g += kGroupsAtOnce) {
    const float* part = t.part + g * t.n * D + col;
    float s = 0.0f;
    if (col < D) {
      uint32_t r = slice;
      for (; r + 7 * 32 < n; r += 8 * 32) {   // eight loads in flight
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = part[(int64_t)(r + i * 32) * D];
        if (t.weight) {
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] *= weight_of<P>(t, r + i * 32, D, col);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) s += v[i];
      }
      for (; r < n; r += 32) s += t.weight ? part[(int64_t)r * D] * weight_of<P>(t, r, D, col) : part[(int64_t)r * D];
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
    }
  }
}

template <typename P>
hipError_t launch_column_sums(SumTasks tasks, int n, hipStream_t s) {
  unsigned at = 0;
  for (int i = 0; i < 3; i++) {
    tasks.first[i] = i < n ? at : 0xffffffffu;
    if (i < n) at += (unsigned)((tasks.t[i].cols + 31) / 32 * (tasks.t[i].groups < kGroupsAtOnce ? tasks.t[i].groups : kGroupsAtOnce));
  }
  column_sums_kernel<P><<<at, 1024, 0, s>>>(tasks);
  return hipGetLastError();
}

}  // namespace
}  // namespace nest
