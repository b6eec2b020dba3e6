// Gated feed-forward block: workspace layout, choice of tiles, dispatch.
#include "blocks_internal.h"

#include <cmath>

namespace nest {
namespace {

// Rows up to which the forward streams the weights through registers
// (gated_few.h).  2048 -> 8192, weights from memory, us, streamed and in tiles:
// 8 rows bf16 24 and 33, 16 rows 28 and 30, 32 rows 37 and 30; float32 45 and
// 75 for one row, 67 and 70 for 16.
constexpr int64_t kFewRows = 16;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Seconds that `groups` workgroups of tiles of side x side and `steps` steps of
// 128 bytes of k take, in rounds of what the LDS lets run at once.  A step of a
// round takes its products' time at the rate a full CU reaches, or what a lone
// workgroup's step takes: its loads' latency (less with four buffers), and for
// float32 the cutting into parts beside the products.  Rates and times are
// fitted to the choices of choose_tile.
double seconds(int64_t groups, int64_t steps, int side, int es) {
  const int i = side == 256 ? 0 : side == 128 ? 1 : 2;
  static constexpr double kRate[2][3] = {{5.2e12, 4.1e12, 2.2e12}, {0.95e12, 0.86e12, 0.59e12}};   // of a CU
  static constexpr double kLone[2][3] = {{0.31e-6, 0.95e-6, 0.44e-6}, {1.9e-6, 1.8e-6, 0.73e-6}};
  static constexpr double kLoneMore[2] = {0.26e-6, 0.70e-6};
  static constexpr int kAtOnce[3] = {1, 2, 5};
  const int f32 = es == 4;
  const double step = 2.0 * side * side * (128 / es) / kRate[f32][i];
  const double lone = side == 64 && groups <= kMoreBuffers ? kLoneMore[f32] : kLone[f32][i];
  auto round = [&](int64_t a_cu) { return (double)steps * (step * a_cu > lone ? step * a_cu : lone); };
  const int64_t full = groups / (256 * kAtOnce[i]), rest = groups % (256 * kAtOnce[i]);
  return (double)full * round(kAtOnce[i]) + (rest ? round(cdiv(rest, 256)) : 0.0);
}

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

// Tiles for up to three products that share a launch and K.  Against every
// tile and split timed at 140 sizes of all five launches (33 to 8192 rows, 160
// to 2048 features, 256 to 8192 hidden; half of them float32) the choice costs
// 0.7% of a call on average, 18% at worst (calls of 20 us); rates fitted to
// those timings would save 0.2%.
TileChoice choose_tile(int n, const int64_t* M, const int64_t* N, int64_t K, int es, bool may_split) {
  TileChoice best{};
  double least = INFINITY;
  const int64_t steps = cdiv(K, 128 / es);
  for (int side = 256; side >= 64; side /= 2) {
    int64_t tiles = 0, size = 0;
    for (int i = 0; i < n; i++) {
      tiles += tiles_along(M[i], side) * tiles_along(N[i], side);
      size += M[i] * N[i];
    }
    for (int splits = 1; splits <= (may_split ? 256 : 1); splits *= 2) {
      if (splits > 1 && steps < 4 * splits) break;   // at least four steps each
      if (tiles * splits * tile_threads(side) > kMostThreads) break;
      double t = seconds(tiles * splits, cdiv(steps, splits), side, es);
      if (splits > 1) t += 4.5e-6 + 8.0 * (double)size * splits / 5e12;   // the partial sums' way to memory and back
      if (t < least) {
        least = t;
        best = {side, splits};
      }
    }
  }
  return best;
}

// Launches of the narrow backward and slices of 32 hidden features in each: the
// least slices in all, then the fewest launches.
void narrow_parts(int ki, int hidden, int& parts, int& slices) {
  const int most = ki <= 2 ? 8 : 4;
  parts = slices = 1 << 20;
  for (int s = most; s >= (ki == 2 ? 2 : 1); s /= 2) {   // one slice of 33 to 64 features: past the registers
    const int n = (hidden + 32 * s - 1) / (32 * s);
    if (n > 1 && s < most / 2) break;   // each launch reads x and dy again
    if (parts == 1 << 20 || n * s < parts * slices) {
      parts = n;
      slices = s;
    }
  }
}

// Whether whole rows stay on the chip (gated_narrow.h): 16-bit rows of at most
// 128 features, where a forward and backward take less time so than in tiles.
//
// Estimated in us from 104 sizes of 32, 64 and 128 features, 128 to 8192 hidden
// and 64 to 640,000 rows, bf16.  Narrow: the weights pass through LDS again for
// every 65536 rows of a forward; a backward takes a launch and a join of its
// workgroups' sums for each part of the hidden features, and each further turn
// of its workgroups.  Tiles: calls of 36 us, or h, g, u and their gradients
// through memory.  A step, narrow and in tiles: 640,000 x 64, 128 179 and 680;
// 65,536 x 64, 1024 254 and 512; 8192 x 64, 512 103 and 49; 8192 x 128, 512 205
// and 55; 64 x 128, 8192 2317 and 42.  The choice costs 0.3% of a step on
// average and 11% at worst; narrow wherever the types and features allow it
// would cost 108%.
bool narrow_rows(int64_t rows, int in, int hidden, int out, int es) {
  if (es != 2 || in > 128 || out > 128 || rows < 64) return false;
  static constexpr double kHidden[4] = {0.028, 0.047, 0.075, 0.1};   // forward, a hidden feature
  static constexpr double kLaunch[4] = {9.5, 13.5, 17.0, 21.0}, kTurn[4] = {2.0, 2.6, 3.5, 4.3};
  const int ki = ((in > out ? in : out) + 31) / 32;
  int parts, slices;
  narrow_parts(ki, hidden, parts, slices);
  const int64_t need = cdiv(rows, 32 * narrow_back_lds(ki, slices).groups), groups = need < 256 ? need : 256;
  const double sums = (double)groups * 3 * slices * 32 * ki * 32 * 4;   // bytes, written and read
  const double forward = hidden * kHidden[ki - 1] * (double)cdiv(rows, 65536);
  const double backward = parts * (kLaunch[ki - 1] + 2.0 * sums / 4.2e6 + (double)(cdiv(need, 256) - 1) * kTurn[ki - 1]);
  const double tiles = 8e-6 * (double)rows * hidden;
  return (forward > 9.0 ? forward : 9.0) + (backward > 19.0 ? backward : 19.0) < (tiles > 36.0 ? tiles : 36.0);
}

GatedLayout gated_layout(int64_t rows, int in, int hidden, int out, int dtype, bool back, bool alone) {
  GatedLayout l{};
  const int es = dtype == NEST_DTYPE_F32 ? 4 : 2, v = 16 / es;
  auto up = [&](int64_t n) { return cdiv(n, v) * v; };
  l.ldx = up(in);
  l.ldh = up(hidden);
  l.ldy = up(out);
  const int64_t kept_bytes = cdiv(rows, 16) * cdiv(l.ldh, 16) * 2048;   // blocks of 16 x 16 g and u
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at = (at + (size_t)bytes + 255) / 256 * 256;
    return o;
  };
  l.narrow = narrow_rows(rows, in, hidden, out, es);
  l.fits = true;
  if (l.narrow) {
    if (!back) return l;
    const int ki = ((in > out ? in : out) + 31) / 32;
    narrow_parts(ki, hidden, l.narrow_parts, l.narrow_slices);
    const int64_t need = cdiv(rows, 32 * narrow_back_lds(ki, l.narrow_slices).groups);
    l.narrow_groups = (int)(need < 256 ? need : 256);
    l.part = take((int64_t)l.narrow_groups * 3 * l.narrow_slices * 32 * ki * 32 * 4);
    if (l.narrow_parts > 1) l.dx_sum = take(cdiv(rows, 32) * 32 * ki * 32 * 4);
    l.bytes = at;
    return l;
  }
  l.h = take(rows * l.ldh * es);
  l.few = !back && rows <= kFewRows;
  if (l.few) {
    l.bytes = at;
    l.kept_bytes = (size_t)kept_bytes;
    return l;
  }
  int64_t part = 0;
  auto partial = [&](const TileChoice& t, int n, const int64_t* M, const int64_t* N) {
    if (t.splits == 1) return;
    int64_t size = 0;
    for (int i = 0; i < n; i++) size += cdiv(M[i] * N[i], kJoinGroup) * kJoinGroup;
    if (size * t.splits * 4 > part) part = size * t.splits * 4;
  };
  if (!back || alone) {
    const int64_t M = rows, N = 2 * (int64_t)hidden;
    l.gate = choose_tile(1, &M, &N, l.ldx, es, false);
    l.fits = l.gate.side != 0;
  }
  if (!back) {
    const int64_t M = rows, N = out;
    l.y = choose_tile(1, &M, &N, l.ldh, es, true);
    partial(l.y, 1, &M, &N);
    l.fits &= l.y.side != 0;
  } else {
    l.gate_back = choose_tile(1, &rows, &l.ldh, out, es, false);
    l.dg = take(rows * l.ldh * es);
    l.du = take(rows * l.ldh * es);
    const int64_t M = rows, N = in;
    l.dx = choose_tile(1, &M, &N, 2 * (int64_t)hidden, es, true);
    // both pairs of a split's sum take the same range of k
    if (l.dx.splits > 1 && cdiv(hidden, 128 / es) < 4 * l.dx.splits) l.dx.splits /= 2;
    partial(l.dx, 1, &M, &N);
    const int64_t WM[3] = {hidden, hidden, out}, WN[3] = {in, in, hidden};
    l.dw = choose_tile(3, WM, WN, rows, es, true);
    partial(l.dw, 3, WM, WN);
    l.fits &= l.gate_back.side != 0 && l.dx.side != 0 && l.dw.side != 0;
    if (alone) l.kept = take(kept_bytes);
    if (l.ldy != out) l.dy = take(rows * l.ldy * es);
  }
  if (l.ldx != in) {
    l.x = take(rows * l.ldx * es);
    l.wg = take(hidden * l.ldx * es);
    l.wu = take(hidden * l.ldx * es);
  }
  if (l.ldh != hidden) l.wd = take(out * l.ldh * es);
  l.part = take(part);
  l.bytes = at;
  l.kept_bytes = (size_t)kept_bytes;
  return l;
}

hipError_t launch_gated_ffn(const GatedParams& p, hipStream_t s, bool back) {
  if (back && p.rows == 0) {
    const size_t es = p.dtype == NEST_DTYPE_F32 ? 4 : 2;
    const size_t up = (size_t)p.in * p.hidden * es, down = (size_t)p.hidden * p.out * es;
    if (hipError_t e = launch_clear(p.dw_gate, up, s); e != hipSuccess) return e;
    if (hipError_t e = launch_clear(p.dw_up, up, s); e != hipSuccess) return e;
    return launch_clear(p.dw_down, down, s);
  }
  if (p.dtype == NEST_DTYPE_F32) return gated_ffn_f32(p, s, back);
  return p.dtype == NEST_DTYPE_F16 ? gated_ffn_f16(p, s, back) : gated_ffn_bf16(p, s, back);
}

}  // namespace nest
