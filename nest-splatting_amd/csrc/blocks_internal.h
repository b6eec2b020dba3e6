// Launch parameters of the decoder block's operators (layer_norm.hip,
// dropout.hip, gated_ffn.hip), shared with the C ABI (abi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/nest_splat.h"

namespace nest {

struct LayerNormParams {
  int64_t rows;
  int cols;
  int dtype, param_dtype;
  float eps;
  const void* x;
  const void* weight;
  const void* bias;    // may be null
  void* y;             // forward
  float* mean;         // [rows]; the forward's may be null
  float* rstd;
  const void* dy;      // backward
  void* dx;
  void* dweight;
  void* dbias;         // may be null
  float* part;         // [layer_norm_partials][2][cols]
};
int layer_norm_partials(int64_t rows, int cols, int dtype);
hipError_t launch_layer_norm(const LayerNormParams& p, hipStream_t s);
hipError_t launch_layer_norm_backward(const LayerNormParams& p, hipStream_t s);

struct DropoutParams {
  int64_t n;
  int dtype;
  const void* x;
  const void* residual;   // may be null
  void* y;
  uint32_t threshold;     // a 16-bit random number below it drops the element
  float scale;
  uint64_t seed, offset;
};
hipError_t launch_dropout(const DropoutParams& p, hipStream_t s);

struct GatedParams {
  int64_t rows;
  int in, hidden, out;
  int dtype, activation;
  const void* x;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  void* y;             // forward
  const void* dy;      // backward
  void* dx;            // each gradient may be null
  void* dw_gate;
  void* dw_up;
  void* dw_down;
  float* kept;         // pre-activations a forward writes or a backward reads, or null
  void* ws;
};

// Tiles of side x side, k split over `splits` workgroups a tile; side 0: no
// tiles that one launch takes.
struct TileChoice {
  int side, splits;
};
inline int64_t tiles_along(int64_t n, int side) { return (n + side - 1) / side; }
constexpr int tile_threads(int side) { return side == 256 ? 512 : 256; }
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1;   // of a launch
// Launches of up to this many workgroups of 64 x 64 tiles, two a CU, take four
// LDS buffers (64 KB) for more loads in flight: forward of 128 rows, 2048 ->
// 8192 bf16, 33 us instead of 39; 1000 rows, 512 -> 2048 f16, 26 instead of 29.
// With more workgroups the others' loads do as well: five of two buffers fit a
// CU, and 1777 x 515, 1365 float32 backward takes 167 us against 188 with four.
constexpr int64_t kMoreBuffers = 512;
constexpr int64_t kJoinGroup = 1024;   // partial sums that a workgroup joins

constexpr int kNarrowLdsBytes = 160 * 1024;
constexpr int kNarrowPad = 16;   // elements past a multiple of 64 bytes: 16-byte reads of 16 rows fall on different banks

// LDS of the forward, in elements: gate and up rows (32 of each in turn), down
// rows, a stage for each wave's stores.
struct NarrowLds {
  int pitch_in, pitch_h, down, stage, total;
};
__host__ __device__ inline NarrowLds narrow_lds(int ki, int hidden, int waves) {
  const int h32 = (hidden + 31) / 32 * 32;
  NarrowLds l;
  l.pitch_in = ki * 32 + kNarrowPad;
  l.pitch_h = h32 + kNarrowPad;
  l.down = 2 * h32 * l.pitch_in;
  l.stage = l.down + ki * 32 * l.pitch_h;
  l.total = l.stage + waves * 16 * (ki * 32 + 8);
  return l;
}

// Waves of a workgroup of the narrow backward, as its registers allow.
__host__ __device__ constexpr int narrow_back_waves(int ki) { return ki <= 2 ? 8 : 4; }

// LDS of the narrow backward, in elements: weights, then for each group of
// waves x, dy [32][row_in] and dg, du [32][row_h]; at its end the groups' sums.
// slices: of 32 hidden features, one a wave.  Rows are a power of two long.
struct NarrowBackLds {
  int groups, row_in, row_h, tiles, tile_stride, total;
};
__host__ __device__ constexpr NarrowBackLds narrow_back_lds(int ki, int slices) {
  NarrowBackLds l{};
  l.groups = narrow_back_waves(ki) / slices;
  l.row_in = ki == 3 ? 128 : ki * 32;
  l.row_h = slices * 32;
  l.tiles = 2 * l.row_h * l.row_in + ki * 32 * l.row_h;
  l.tile_stride = 2 * 32 * l.row_in + 2 * 32 * l.row_h;
  l.total = l.tiles + l.groups * l.tile_stride;
  const int sums = l.groups > 1 ? slices * 12 * ki * 256 * 2 : 0;   // float32: two elements each
  if (sums > l.total) l.total = sums;
  return l;
}

// What a call's sizes fix: row lengths (rounded up to 16 bytes), the
// workspace's parts (byte offsets) and each product's tiles.
struct GatedLayout {
  int64_t ldx, ldh, ldy;
  size_t h, dg, du, kept, x, wg, wu, wd, dy, part;
  size_t bytes, kept_bytes;
  TileChoice gate, gate_back, y, dx, dw;
  bool fits;                  // in launches
  bool narrow;                // gated_narrow.h
  size_t dx_sum;              // of its backward: sums of dx between launches,
  int narrow_parts, narrow_slices;   // launches, and slices of 32 hidden features in each
  bool few;                   // gated_few.h (forward)
  int narrow_groups;          // workgroups of its backward
};
GatedLayout gated_layout(int64_t rows, int in, int hidden, int out, int dtype, bool backward, bool alone);
hipError_t launch_gated_ffn(const GatedParams& p, hipStream_t s, bool backward);
hipError_t gated_ffn_f32(const GatedParams& p, hipStream_t s, bool backward);
hipError_t gated_ffn_f16(const GatedParams& p, hipStream_t s, bool backward);
hipError_t gated_ffn_bf16(const GatedParams& p, hipStream_t s, bool backward);

}  // namespace nest
