// The calls of a gated feed-forward block for one element type: included by
// gated_ffn_f32.hip, gated_ffn_f16.hip and gated_ffn_bf16.hip.
#pragma once

#include "gated_few.h"
#include "gated_narrow.h"
#include "gated_tiles.h"

namespace nest {
namespace {

template <typename T>
hipError_t gated_forward(const GatedParams& p, hipStream_t s) {
  const GatedLayout l = gated_layout(p.rows, p.in, p.hidden, p.out, p.dtype, false, false);
  if constexpr (sizeof(T) == 2)
    if (l.narrow) return launch_narrow_forward<T>(p, s);
  if (l.few) return launch_few_forward<T>(p, l, s);
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  Operands<T> o;
  if (hipError_t e = pad_operands(p, l, ws, false, o, s); e != hipSuccess) return e;
  T* h = reinterpret_cast<T*>(ws + l.h);
  Gate<T> g{o.x, o.wg, o.wu, l.ldx, (int)p.rows, p.hidden, l.ldh, h, p.kept, p.activation, 0, 0};
  if (hipError_t e = launch_gate(g, l.gate, s); e != hipSuccess) return e;
  Products<T> y{};
  y.n = 1;
  y.p[0] = {h, o.wd, nullptr, nullptr, l.ldh, l.ldh, (int)p.rows, p.out, l.ldh, static_cast<T*>(p.y)};
  y.part = reinterpret_cast<float*>(ws + l.part);
  return launch_products<T, true, true>(y, l.y, s);
}

template <typename T>
hipError_t gated_backward(const GatedParams& p, hipStream_t s) {
  const GatedLayout l = gated_layout(p.rows, p.in, p.hidden, p.out, p.dtype, true, p.kept == nullptr);
  if constexpr (sizeof(T) == 2)
    if (l.narrow) return launch_narrow_backward<T>(p, l, s);
  const bool alone = p.kept == nullptr;
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  T *h = reinterpret_cast<T*>(ws + l.h), *dg = reinterpret_cast<T*>(ws + l.dg), *du = reinterpret_cast<T*>(ws + l.du);
  Operands<T> o;
  if (hipError_t e = pad_operands(p, l, ws, true, o, s); e != hipSuccess) return e;
  float* kept = p.kept;
  if (alone) {
    kept = reinterpret_cast<float*>(ws + l.kept);
    Gate<T> g{o.x, o.wg, o.wu, l.ldx, (int)p.rows, p.hidden, l.ldh, nullptr, kept, p.activation, 0, 0};
    if (hipError_t e = launch_gate(g, l.gate, s); e != hipSuccess) return e;
  }
  GateBackward<T> b{o.dy, o.wd, l.ldy, l.ldh, (int)p.rows, p.out, p.hidden, kept, h, dg, du, p.activation, 0, 0};
  if (hipError_t e = launch_gate_backward(b, l.gate_back, s); e != hipSuccess) return e;
  if (p.dx) {
    Products<T> q{};
    q.n = 1;
    q.p[0] = {dg, o.wg, du, o.wu, l.ldh, l.ldx, (int)p.rows, p.in, p.hidden, static_cast<T*>(p.dx)};
    q.part = reinterpret_cast<float*>(ws + l.part);
    if (hipError_t e = launch_products<T, true, false>(q, l.dx, s); e != hipSuccess) return e;
  }
  Products<T> w{};
  if (p.dw_gate) w.p[w.n++] = {dg, o.x, nullptr, nullptr, l.ldh, l.ldx, p.hidden, p.in, p.rows, static_cast<T*>(p.dw_gate)};
  if (p.dw_up) w.p[w.n++] = {du, o.x, nullptr, nullptr, l.ldh, l.ldx, p.hidden, p.in, p.rows, static_cast<T*>(p.dw_up)};
  if (p.dw_down) w.p[w.n++] = {o.dy, h, nullptr, nullptr, l.ldy, l.ldh, p.out, p.hidden, p.rows, static_cast<T*>(p.dw_down)};
  if (!w.n) return hipSuccess;
  w.part = reinterpret_cast<float*>(ws + l.part);
  return launch_products<T, false, false>(w, l.dw, s);
}

}  // namespace
}  // namespace nest
