"""64-bit formulas of the decoder block's operators, each with a bound of how
far a 32-bit computation that rounds its stated intermediates may be off.

The bounds are first-order error analysis, element by element: a sum of n
terms is off by at most gamma(n) times the sum of the terms' magnitudes,
gamma(n) = (n + 8) 2^-24; a value rounded to type T by u(T) times itself plus
half of T's smallest step."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
F32 = 2.0 ** -24


def gamma(n):
    return (n + 8) * F32


def rounded(v, err, dtype):
    """The bound after v, off by err, is rounded to dtype."""
    return err + UNIT[dtype] * (v.abs() + err) + TINY[dtype]


def check(got, want, bound, what):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    bad = ~(d <= bound)  # NaN counts as wrong
    assert not bad.any(), f"{what}: {int(bad.sum())} of {d.numel()} past the bound, worst {float((d / bound).nan_to_num(1e9).max()):.3g} times it"


def norm(x, w, b, eps, dy=None):
    """{name: (value, bound)} of y, and of dx, dw, db where dy is given."""
    T, P = x.dtype, w.dtype
    x, w = x.double(), w.double()
    N, D = x.shape
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    h = (x - mean) * rstd
    e_mean = gamma(D) * x.abs().mean(1, keepdim=True)
    r_rstd = 0.5 * ((e_mean * rstd) ** 2 + 2 * F32 * (x.abs().amax(1, keepdim=True) * rstd) + gamma(D)) + 4 * F32
    e_h = rstd * (e_mean + F32 * x.abs()) + h.abs() * (r_rstd + 4 * F32)
    y = h * w + b
    out = {"y": (y, rounded(y, e_h * w.abs() + 2 * F32 * ((h * w).abs() + b.abs()), T))}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    a, c = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    e_a = gamma(D) * g.abs().mean(1, keepdim=True)
    e_c = gamma(D) * (g * h).abs().mean(1, keepdim=True) + (g.abs() * e_h).mean(1, keepdim=True)
    dx = rstd * (g - a - h * c)
    size = g.abs() + a.abs() + (h * c).abs()
    e_dx = rstd * (e_a + e_h * c.abs() + h.abs() * e_c + 4 * F32 * size) + dx.abs() * (r_rstd + 4 * F32)
    out["dx"] = (dx, rounded(dx, e_dx, T))
    dw, db = (dy * h).sum(0), dy.sum(0)
    out["dw"] = (dw, rounded(dw, gamma(N) * (dy * h).abs().sum(0) + (dy.abs() * e_h).sum(0), P))
    out["db"] = (db, rounded(db, gamma(N) * dy.abs().sum(0), P))
    return out


def act(g, kind):
    """(value, slope, a bound of the second derivative)."""
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double(), 0.0
    if kind == "silu":
        q = torch.sigmoid(g)
        return g * q, q * (1 + g * (1 - q)), 0.5
    q = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * q, q + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 0.8


def ffn(x, wg, wu, wd, kind, dy=None):
    """{name: (value, bound)} of y, and of dx, dw_gate, dw_up, dw_down where dy is given."""
    T = x.dtype
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    N, I = x.shape
    H, O = wg.shape[0], wd.shape[0]
    g, u = x @ wg.T, x @ wu.T
    e_g, e_u = gamma(I) * (x.abs() @ wg.abs().T), gamma(I) * (x.abs() @ wu.abs().T)
    a, s, curve = act(g, kind)
    calc = 2.0 ** -19  # exp or erf, a division and a few products, of g's size
    e_a = 1.2 * e_g + calc * a.abs() + 2.0 ** -22 * g.abs()
    h = a * u
    e_h = rounded(h, e_a * u.abs() + a.abs() * e_u + e_a * e_u, T)
    y = h @ wd.T
    out = {"y": (y, rounded(y, e_h @ wd.abs().T + gamma(H) * (h.abs() @ wd.abs().T), T))}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ wd
    e_dh = gamma(O) * (dy.abs() @ wd.abs())
    e_s = curve * e_g + calc * (1 + g.abs()) * (0 if kind == "relu" else 1)
    if kind == "relu":
        e_s = (g.abs() <= e_g).double()  # the sign itself may be off
    dg, du = dh * u * s, dh * a
    e_dg = rounded(dg, e_dh * (u * s).abs() + (dh * s).abs() * e_u + (dh * u).abs() * e_s + 4 * F32 * dg.abs(), T)
    e_du = rounded(du, e_dh * a.abs() + dh.abs() * e_a + 4 * F32 * du.abs(), T)
    dx = dg @ wg + du @ wu
    out["dx"] = (dx, rounded(dx, e_dg @ wg.abs() + e_du @ wu.abs() + gamma(2 * H) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()), T))
    for name, d, e in (("dw_gate", dg, e_dg), ("dw_up", du, e_du)):
        v = d.T @ x
        out[name] = (v, rounded(v, e.T @ x.abs() + gamma(N) * (d.abs().T @ x.abs()), T))
    v = dy.T @ h
    out["dw_down"] = (v, rounded(v, dy.abs().T @ e_h + gamma(N) * (dy.abs().T @ h.abs()), T))
    return out


def philox_halves(blocks, seed, offset):
    """The eight 16-bit halves of each counter's Philox 4x32-10 block, in whole numbers."""
    out = []
    for c in blocks:
        v = [c & 0xFFFFFFFF, c >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            p0, p1 = 0xD2511F53 * v[0], 0xCD9E8D57 * v[2]
            v = [(p1 >> 32) ^ v[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ v[3] ^ k[1], p0 & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for w in v:
            out += [w & 0xFFFF, w >> 16]
    return out


def dropped(n, p, seed, offset, first_block=0):
    t = math.floor(p * 65536 + 0.5)
    halves = philox_halves(range(first_block, first_block + (n + 7) // 8), seed, offset)[:n]
    return torch.tensor(halves) < t, (65536.0 / (65536 - t) if t < 65536 else 0.0)
