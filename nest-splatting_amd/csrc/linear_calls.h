// The calls of a dense layer for one element type: included by linear_f32.hip,
// linear_f16.hip and linear_bf16.hip.
#pragma once

#include "linear_narrow.h"
#include "linear_narrow_f32.h"
#include "linear_tiles.h"

namespace nest {
namespace {

// Operands whose rows are no multiple of 16 bytes, copied to rows that are.
template <typename T>
hipError_t pad_rows(const T*& x, int64_t x_rows, T* x_to, const T*& w, int64_t w_rows, T* w_to, int len, int64_t ld, hipStream_t s) {
  Pads<T> q{};
  int n = 0;
  int64_t most = 0;
  auto add = [&](const T*& from, int64_t rows, T* to) {
    if (!to) return;
    q.from[n] = from;
    q.to[n] = to;
    q.rows[n] = rows;
    q.n[n] = len;
    q.ld[n++] = (int)ld;
    most = rows * ld > most ? rows * ld : most;
    from = to;
  };
  add(x, x_rows, x_to);
  add(w, w_rows, w_to);
  if (n) {
    const int64_t need = (most / Vec16<T>::kN + 255) / 256;
    pad_kernel<T><<<dim3((unsigned)(need < 4096 ? need : 4096), n), 256, 0, s>>>(q);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t linear_forward(const LinearParams& p, hipStream_t s) {
  const LinearLayout l = linear_layout(p, false);
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w);
  const Epilogue<T> ep{static_cast<const T*>(p.bias), static_cast<const T*>(p.residual), static_cast<T*>(p.y), p.kept, p.slope_bytes,
                       p.activation, p.out};
  if constexpr (sizeof(T) == 2) {
    if (l.narrow) return launch_narrow_layer<T>(p, s);
  } else {
    if (l.narrow) return launch_narrow_f32<T>(p, ep, s);
  }
  if (l.few) {
    const Few<T> few{x, w, nullptr, p.in, (int)p.rows, p.out, p.in, static_cast<T*>(p.y), p.out, nullptr, 0};
    return launch_few<T, false>(few, s, FinishSum<T>{ep});
  }
  if (l.ldx != p.in)
    if (hipError_t e = pad_rows(x, p.rows, reinterpret_cast<T*>(ws + l.x), w, p.out, reinterpret_cast<T*>(ws + l.w), p.in, l.ldx, s); e != hipSuccess)
      return e;
  LinearTiles<T> t{x, w, l.ldx, (int)p.rows, p.out, ep, (int)tiles_along(p.rows, l.y.side), (int)tiles_along(p.out, l.y.side), l.y.splits,
                   l.y.splits > 1 ? reinterpret_cast<float*>(ws + l.part) : nullptr};
  const unsigned grid = (unsigned)((int64_t)t.tiles_m * t.tiles_n * t.splits);
  with_tile(l.y.side, grid, [&](auto c) {
    typedef decltype(c) C;
    linear_tile_kernel<T, C><<<grid, C::NT, 0, s>>>(t);
  });
  if (l.y.splits > 1) {
    const int64_t need = (p.rows * ((p.out + Vec16<T>::kN - 1) / Vec16<T>::kN) + 255) / 256;
    linear_join_kernel<T><<<(unsigned)(need < 65536 ? need : 65536), 256, 0, s>>>(t);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t linear_backward(const LinearParams& p, hipStream_t s) {
  const LinearLayout l = linear_layout(p, true);
  if constexpr (sizeof(T) == 2) {
    if (l.narrow) return launch_narrow_layer_backward<T>(p, l, s);
  } else {
    if (l.narrow) return launch_narrow_f32_backward<T>(p, l, s);
  }
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  const bool products = p.dx || p.dw;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *dz = static_cast<const T*>(p.dy);
  T* const made = l.copy_dz && products ? reinterpret_cast<T*>(ws + l.dz) : nullptr;
  if (made || p.db) {
    const SlopeRows<T> q{dz, p.kept, p.slope_bytes, p.rows, p.out, l.ldz, made, p.db ? reinterpret_cast<float*>(ws + l.sums) : nullptr};
    if (hipError_t e = launch_slopes(q, l.sum_rows, s); e != hipSuccess) return e;
    if (p.db) {
      SumTasks t{};
      t.t[0] = {q.part, l.sum_rows, 1, p.out, nullptr, nullptr, p.db, nullptr};
      if (hipError_t e = launch_column_sums<T>(t, 1, s); e != hipSuccess) return e;
    }
    if (made) dz = made;
  }
  if (!products) return hipSuccess;
  if (p.codes && p.dw) {
    T* to = reinterpret_cast<T*>(ws + l.x);
    if (hipError_t e = launch_unpack8(p.rows, p.in, p.dtype, p.codes, p.steps, to, l.ldx, s); e != hipSuccess) return e;
    x = to;
  }
  if (l.ldx != p.in) {
    T* const x_to = p.dw && !p.codes ? reinterpret_cast<T*>(ws + l.x) : nullptr;
    T* const w_to = p.dx ? reinterpret_cast<T*>(ws + l.w) : nullptr;
    if (hipError_t e = pad_rows(x, p.rows, x_to, w, p.out, w_to, p.in, l.ldx, s); e != hipSuccess) return e;
  }
  Products<T> q{};
  q.n = 1;
  q.part = reinterpret_cast<float*>(ws + l.part);
  if (p.dx) {
    q.p[0] = {dz, w, nullptr, nullptr, l.ldz, l.ldx, (int)p.rows, p.in, p.out, static_cast<T*>(p.dx)};
    if (hipError_t e = launch_products<T, true, false>(q, l.dx, s); e != hipSuccess) return e;
  }
  if (!p.dw) return hipSuccess;
  q.part = reinterpret_cast<float*>(ws + l.part);
  q.p[0] = {dz, x, nullptr, nullptr, l.ldz, l.ldx, p.out, p.in, p.rows, static_cast<T*>(p.dw)};
  return launch_products<T, false, false>(q, l.dw, s);
}

}  // namespace
}  // namespace nest
