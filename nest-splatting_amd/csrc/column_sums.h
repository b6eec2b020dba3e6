// Sums of partial rows by column, for the gradients of what rows share
// (residual_norm.hip, linear_calls.h).
#pragma once

#include "vec_io.h"

namespace nest {
namespace {

// For each of `groups` groups the sum of n rows (below 2^32): out0 = the sum
// times mul0 and out1 times mul1 by column.
struct SumTask {
  const float* part;
  int64_t n, groups;
  int cols;
  const void *mul0, *mul1;
  void *out0, *out1;
};
// Of a task; a workgroup takes every 4096th. 3 tasks of 256 workgroups across
// stay under 2^32 threads a launch.
constexpr int64_t kGroupsAtOnce = 4096;
struct SumTasks {
  SumTask t[3];
  unsigned first[3];   // workgroup of each task
};

// Groups of so few rows go to a slice of a workgroup each.
constexpr int64_t kFewSummed = 16;
inline int64_t groups_at_once(const SumTask& t) { return t.n <= kFewSummed ? 32 : 1; }

// 32 columns a workgroup, 32 slices of a group's rows, joined in LDS in their
// order, or of few rows 32 groups (100,000 groups of one row of 64 columns: 389
// us a group at a time).
template <typename P>
__global__ __launch_bounds__(1024) void column_sums_kernel(SumTasks tasks) {
  __shared__ float lds[32][33];
  const int which = blockIdx.x >= tasks.first[2] ? 2 : blockIdx.x >= tasks.first[1] ? 1 : 0;
  const SumTask& t = tasks.t[which];
  const int64_t D = t.cols;
  const unsigned across = (unsigned)((D + 31) / 32), id = blockIdx.x - tasks.first[which];
  const int col = (int)(id % across) * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  const uint32_t n = (uint32_t)t.n;
  auto put = [&](int64_t g, float v) {
    auto out = [&](void* to, const void* mul) {
      if (to) static_cast<P*>(to)[g * D + col] = from_f32<P>(mul ? v * to_f32(static_cast<const P*>(mul)[col]) : v);
    };
    out(t.out0, t.mul0);
    out(t.out1, t.mul1);
  };
  if (n <= kFewSummed) {
    for (int64_t g = (int64_t)(id / across) * 32 + slice; g < t.groups; g += kGroupsAtOnce * 32) {
      if (col >= D) break;
      float s = 0.0f;
      for (uint32_t r = 0; r < n; r++) s += t.part[(g * n + r) * D + col];
      put(g, s);
    }
    return;
  }
  for (int64_t g = id / across; g < t.groups; g += kGroupsAtOnce) {
    const float* part = t.part + g * t.n * D + col;
    float s = 0.0f;
    if (col < D) {
      uint32_t r = slice;
      for (; r + 7 * 32 < n; r += 8 * 32) {   // eight loads in flight
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = part[(int64_t)(r + i * 32) * D];
#pragma unroll
        for (int i = 0; i < 8; i++) s += v[i];
      }
      for (; r < n; r += 32) s += part[(int64_t)r * D];
    }
    __syncthreads();   // the last group's sums are all read
    lds[slice][threadIdx.x & 31] = s;
    __syncthreads();
    if (slice == 0 && col < D) {
      float all = 0.0f;
#pragma unroll
      for (int r = 0; r < 32; r++) all += lds[r][threadIdx.x];
      put(g, all);
    }
  }
}

template <typename P>
hipError_t launch_column_sums(SumTasks tasks, int n, hipStream_t s) {
  unsigned at = 0;
  for (int i = 0; i < 3; i++) {
    tasks.first[i] = i < n ? at : 0xffffffffu;
    if (i >= n) continue;
    const int64_t need = (tasks.t[i].groups + groups_at_once(tasks.t[i]) - 1) / groups_at_once(tasks.t[i]);
    at += (unsigned)((tasks.t[i].cols + 31) / 32 * (need < kGroupsAtOnce ? need : kGroupsAtOnce));
  }
  column_sums_kernel<P><<<at, 1024, 0, s>>>(tasks);
  return hipGetLastError();
}

}  // namespace
}  // namespace nest
