// Launch parameters of a residual block's operators (linear*.hip, pack8.hip,
// residual_norm.hip, embedding.hip), shared with the C ABI (abi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/nest_splat.h"
#include "blocks_internal.h"

namespace nest {

// ---- residual_norm.hip ----

struct ResidualNormParams {
  int64_t rows;
  int cols;
  int dtype, param_dtype;
  float scale, eps;
  const void* x;
  const void* h;          // null: r is x and is not written
  const void* gate;       // [gates][cols] or null
  int64_t gates;          // rows / gates rows share one
  const void* post;       // [cols] or null: h is not normed
  const void* pre;        // [cols] or null: no y
  void* r;                // forward's result, backward's operand (x where h is null)
  void* y;
  float* rstd_post;       // [rows]; the forward's may be null
  float* rstd_pre;
  const void* dr;         // backward; null: zero
  const void* dy;         // null: zero
  void* dx;
  void* dh;               // with h
  void* dgate;            // with gate
  void* dpost;            // with post
  void* dpre;             // with pre
  float* ws;
};
constexpr int kResidualNormCols = 8192;   // a workgroup holds one row in registers
size_t residual_norm_ws_bytes(int64_t rows, int cols, int dtype, int64_t gates);
hipError_t launch_residual_norm(const ResidualNormParams& p, hipStream_t s);
hipError_t launch_residual_norm_backward(const ResidualNormParams& p, hipStream_t s);

// ---- embedding.hip ----

struct EmbeddingParams {
  int64_t rows;           // of ids
  int cols;
  int64_t table_rows;     // an id outside [0, table_rows) has no row
  int dtype;
  bool wide_ids;          // int64, else int32
  const void* ids;
  float scale;
  const void* table;      // forward
  const void* residual;   // or null
  void* y;
  const void* dy;         // backward
  void* dtable;
  void* ws;
};
size_t embedding_ws_bytes(int64_t rows, int cols, int64_t table_rows, int dtype);
hipError_t launch_embedding(const EmbeddingParams& p, hipStream_t s);
hipError_t launch_embedding_backward(const EmbeddingParams& p, hipStream_t s);

// ---- pack8.hip ----

constexpr int kPackGroup = 32;          // values of a row that share a step
inline int64_t pack_groups(int cols) { return (cols + kPackGroup - 1) / kPackGroup; }
hipError_t launch_pack8(int64_t rows, int cols, int dtype, const void* x, int8_t* codes, uint8_t* steps, hipStream_t s);
// Rows of y are ldy values long, those from cols on zero.
hipError_t launch_unpack8(int64_t rows, int cols, int dtype, const int8_t* codes, const uint8_t* steps, void* y, int64_t ldy,
                          hipStream_t s);

// ---- linear*.hip ----

struct LinearParams {
  int64_t rows;
  int in, out;
  int dtype, activation;
  int slope_bytes;         // of a kept slope
  const void* x;
  const int8_t* codes;     // a backward's x in 8 bits, or null
  const uint8_t* steps;
  const void* w;
  const void* bias;        // or null
  const void* residual;    // or null
  void* y;                 // forward
  void* kept;              // slopes a forward writes, or null, and a backward reads
  const void* dy;          // backward
  void* dx;                // each gradient may be null
  void* dw;
  void* db;
  void* ws;
};

// What a call's sizes fix: row lengths (rounded up to 16 bytes), the
// workspace's parts (byte offsets) and each product's tiles.
struct LinearLayout {
  int64_t ldx, ldz;
  size_t x, w, dz, sums, part, bytes;
  TileChoice y, dx, dw;
  bool narrow;             // linear_narrow.h, linear_narrow_f32.h
  bool few;                // gated_few.h (forward)
  bool fits;               // in launches
  bool copy_dz;            // the backward makes dz; it is dy itself otherwise
  int sum_rows;            // workgroups that gather db
};
LinearLayout linear_layout(const LinearParams& p, bool backward);
// Rows that stay on the chip; a backward makes their slopes again from x and
// the bias unless they are kept in 8 bits.
inline bool linear_narrow(int in, int out, int dtype) { return dtype != NEST_DTYPE_F32 && in <= 128 && out <= 128; }
// Workgroups of their backward that run on a CU at once, by 32s of features in
// and out and whether anything is kept in 8 bits: as the registers allow.
constexpr int kNarrowBackRows = 64;   // of a workgroup's turn
constexpr int narrow_groups_cu(int ki, int ko, bool saved) {
  const int size = ki + ko + (saved ? 1 : 0);
  return size <= 4 ? 4 : size <= 5 ? 3 : ki + ko <= 6 ? 2 : 1;
}
// float32 rows that stay on the chip (linear_narrow_f32.h); their slopes are
// kept.
inline bool linear_narrow_f32(int in, int out, int dtype) { return dtype == NEST_DTYPE_F32 && in <= 64 && out <= 64; }
// Workgroups of their backward on a CU, by 16s of features in and out: as the
// registers allow.
constexpr int narrow_f32_groups(int ki, int ko) { return ki * ko <= 4 && ko < 4 ? 4 : ki * ko <= 9 ? 3 : 2; }
int linear_slope_bytes(int in, int out, int dtype, int activation, bool save8);
hipError_t launch_linear(const LinearParams& p, hipStream_t s, bool backward);
hipError_t linear_f32(const LinearParams& p, hipStream_t s, bool backward);
hipError_t linear_f16(const LinearParams& p, hipStream_t s, bool backward);
hipError_t linear_bf16(const LinearParams& p, hipStream_t s, bool backward);

TileChoice choose_tile(int n, const int64_t* M, const int64_t* N, int64_t K, int es, bool may_split);   // gated_ffn.hip

}  // namespace nest
