// Dense layer: workspace layout, choice of tiles, dispatch.
#include "residual_internal.h"

namespace nest {
namespace {

// Rows up to which the forward streams the weights through registers, as
// gated_ffn does.  us of a call so and in tiles, weights from memory: bf16, 2
// rows of 8192 -> 2048 11.4 and 13.8, 16 11.6 and 13.8, 16 of 2048 -> 8192 9.8 and
// 10.9; float32, 2 of 2048 -> 8192 15.9 and 27, 16 24.5 and 25.3, 16 of 8192 ->
// 2048 29.5 and 27, of 2048 -> 2048 9.1 and 13.9.  One row of 2048 -> 8192 takes
// 8.8 us on the GPU: 33.6 MB of weights at 3.8 TB/s.
constexpr int64_t kFewRows = 16;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

__global__ __launch_bounds__(256) void clear_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

hipError_t launch_clear(void* p, size_t bytes, hipStream_t s) {
  if (!p) return hipSuccess;
  const int64_t n = (int64_t)bytes / 2, need = cdiv(n, 256);
  clear_kernel<<<(unsigned)(need < 65536 ? need : 65536), 256, 0, s>>>(static_cast<uint16_t*>(p), n);
  return hipGetLastError();
}

}  // namespace

int linear_slope_bytes(int in, int out, int dtype, int activation, bool save8) {
  if (activation == NEST_ACT_NONE || (!save8 && linear_narrow(in, out, dtype))) return 0;
  if (activation == NEST_ACT_RELU) return 1;
  return (save8 ? 1 : 2) * (dtype == NEST_DTYPE_F32 ? 2 : 1);
}

LinearLayout linear_layout(const LinearParams& p, bool back) {
  LinearLayout l{};
  const int es = p.dtype == NEST_DTYPE_F32 ? 4 : 2, v = 16 / es;
  l.ldx = cdiv(p.in, v) * v;
  l.ldz = cdiv(p.out, v) * v;
  l.fits = true;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at = (at + (size_t)bytes + 255) / 256 * 256;
    return o;
  };
  const bool narrow_f32 = linear_narrow_f32(p.in, p.out, p.dtype);
  l.narrow = narrow_f32 || linear_narrow(p.in, p.out, p.dtype);
  if (l.narrow) {
    if (!back) return l;
    // as many workgroups as run at once, by LDS and registers
    auto blocks = [](int v, int of) { return (v + of - 1) / of; };
    const int a_cu = narrow_f32 ? narrow_f32_groups(blocks(p.in, 16), blocks(p.out, 16))
                                : narrow_groups_cu(blocks(p.in, 32), blocks(p.out, 32), p.slope_bytes || p.codes);
    const int64_t turns = cdiv(p.rows, kNarrowBackRows);
    l.sum_rows = (int)(turns < 256 * a_cu ? turns : 256 * a_cu);
    l.sums = take(l.sum_rows * (int64_t)p.out * 4);
    l.part = take(l.sum_rows * (int64_t)p.out * p.in * 4);
    l.bytes = at;
    return l;
  }
  int64_t part = 0;
  auto partial = [&](const TileChoice& t, int64_t M, int64_t N) {
    const int64_t bytes = t.splits * cdiv(M * N, kJoinGroup) * kJoinGroup * 4;
    if (t.splits > 1 && bytes > part) part = bytes;
    l.fits &= t.side != 0;
  };
  if (!back) {
    l.few = p.rows <= kFewRows;
    if (l.few) return l;
    const int64_t M = p.rows, N = p.out;
    l.y = choose_tile(1, &M, &N, l.ldx, es, true);
    partial(l.y, M, N);
  } else {
    const int64_t M = p.rows, I = p.in, O = p.out;
    l.dx = choose_tile(1, &M, &I, O, es, true);
    partial(l.dx, M, I);
    l.dw = choose_tile(1, &O, &I, M, es, true);
    partial(l.dw, O, I);
    l.copy_dz = p.slope_bytes != 0 || l.ldz != p.out;
    if (l.copy_dz) l.dz = take(M * l.ldz * es);
    const int64_t vecs = l.ldz / v;
    int64_t lanes = 1;
    while (lanes < vecs && lanes < 64) lanes *= 2;
    const int64_t turns = cdiv(M, 256 / lanes * 4), most = cdiv(2048, cdiv(vecs, lanes));
    l.sum_rows = (int)(turns < most ? turns : most);
    l.sums = take(l.sum_rows * O * 4);
  }
  if (l.ldx != p.in || p.codes) l.x = take(p.rows * l.ldx * es);
  if (l.ldx != p.in) l.w = take(p.out * l.ldx * es);
  l.part = take(part);
  l.bytes = at;
  return l;
}

hipError_t launch_linear(const LinearParams& p, hipStream_t s, bool back) {
  if (back && p.rows == 0) {
    const size_t es = p.dtype == NEST_DTYPE_F32 ? 4 : 2;
    if (hipError_t e = launch_clear(p.dw, (size_t)p.in * p.out * es, s); e != hipSuccess) return e;
    return launch_clear(p.db, (size_t)p.out * es, s);
  }
  if (p.dtype == NEST_DTYPE_F32) return linear_f32(p, s, back);
  return p.dtype == NEST_DTYPE_F16 ? linear_f16(p, s, back) : linear_bf16(p, s, back);
}

}  // namespace nest
