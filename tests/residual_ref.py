"""64-bit formulas of the residual block's operators, each with a bound of how
far a 32-bit computation that rounds its stated intermediates may be off (see
block_ref.py for the analysis that the bounds follow)."""
import torch

import block_ref as R

F32, gamma, rounded, check = R.F32, R.gamma, R.rounded, R.check
FINE, COARSE = 26000.0, 200.0
CALC = 2.0 ** -19   # exp or erf, a division and a few products, of the argument's size


def act(z, kind):
    return (z, torch.ones_like(z), 0.0) if kind is None else R.act(z, kind)


def slope_step(dtype, kind, save8):
    """The step that slopes are kept in, 0 for exact."""
    if kind in (None, "relu"):
        return 0.0
    if dtype is torch.float32:
        return 1 / FINE if save8 else 0.0
    return 1 / COARSE if save8 else 1 / FINE


def pre_activation(x, w, b):
    """(z, how far it may be off)."""
    x, w = x.double(), w.double()
    z, size = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, gamma(x.shape[1] + 1) * size


def linear(x, w, b, kind, r=None, dy=None, save8=False, packed=None):
    """{name: (value, bound)} of y, and of dx, dw, db where dy is given; packed: the values that x in 8 bits stands for."""
    T = x.dtype
    z, e_z = pre_activation(x, w, b)
    N, O = z.shape
    a, s, curve = act(z, kind)
    smooth = kind in ("silu", "gelu")
    e_a = 1.2 * e_z + ((CALC * a.abs() + 2.0 ** -22 * z.abs()) if smooth else 0)
    y = a if r is None else a + r.double()
    out = {"y": (y, rounded(y, e_a + 2 * F32 * (a.abs() + y.abs()), T))}
    if dy is None:
        return out
    w64, dy = w.double(), dy.double()
    x64 = (x if packed is None else packed).double()
    if smooth:
        step = slope_step(T, kind, save8)
        e_s = curve * e_z + CALC * (1 + z.abs()) + step / 2 + 4 * F32   # a code is the nearest to the slope that was computed
    elif kind == "relu":
        e_s = (z.abs() <= e_z).double()   # the sign itself may be off
    else:
        e_s = torch.zeros_like(z)
    dz = dy * s
    e_exact = dy.abs() * e_s + 2 * F32 * dz.abs()
    e_dz = rounded(dz, e_exact, T) if kind is not None else torch.zeros_like(dz)
    dx = dz @ w64
    out["dx"] = (dx, rounded(dx, e_dz @ w64.abs() + gamma(O) * ((dz.abs() + e_dz) @ w64.abs()), T))
    dw = dz.T @ x64
    out["dw"] = (dw, rounded(dw, e_dz.T @ x64.abs() + gamma(N) * ((dz.abs() + e_dz).T @ x64.abs()), T))
    db = dz.sum(0)
    out["db"] = (db, rounded(db, e_exact.sum(0) + gamma(N) * (dz.abs() + e_exact).sum(0), T))
    return out


def pack(x):
    """(codes, steps, values) of rows in 8 bits, by whole-number arithmetic on exponents."""
    v = x.double()
    D = v.shape[-1]
    groups = torch.nn.functional.pad(v, (0, -D % 32)).reshape(*v.shape[:-1], -1, 32)
    bad = ~torch.isfinite(groups).all(-1)
    safe = torch.where(bad[..., None], 0.0, groups)
    e = (torch.frexp(safe.abs().amax(-1))[1] - 1).clamp(min=-126)
    e = torch.where(safe.abs().amax(-1) == 0, -126, e)
    step = ((e.long() - 6 + 1023) << 52).view(torch.float64)[..., None]   # 2^(e - 6) by its bits: a power function may be off by its last one
    codes = torch.round(safe / step).clamp(-127, 127)
    values = torch.where(bad[..., None], float("nan"), codes * step)
    flat = lambda t: t.reshape(*v.shape[:-1], -1)[..., :D]
    return flat(codes).to(torch.int8), torch.where(bad, 255, e + 126).to(torch.uint8), flat(values).to(x.dtype)


def gate_rows(gate, rows):
    """gate [G, D] as one row for each of `rows`."""
    return torch.ones(1, 1, dtype=torch.float64, device=gate.device) if gate is None else gate.double().repeat_interleave(rows // gate.shape[0], 0)


def inv_rms(v, eps):
    return 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def residual_norm_r(x, h, gate, post, scale, eps):
    """(r, bound) over rows [N, D], gate [G, D] or None."""
    T, D = x.dtype, x.shape[1]
    x, h = x.double(), h.double()
    a, rel = (1.0, 0.0) if post is None else (inv_rms(h, eps), 0.5 * gamma(D) + 4 * F32)
    t = h * a * (1.0 if post is None else post.double())
    gt = t if gate is None else t * gate_rows(gate, x.shape[0])
    r = scale * x + gt
    return r, rounded(r, gt.abs() * (rel + 6 * F32) + 4 * F32 * ((scale * x).abs() + gt.abs()), T)


def residual_norm_y(r, pre, eps):
    """(y, bound) from r as it is stored."""
    y = r.double() * inv_rms(r.double(), eps) * pre.double()
    return y, rounded(y, y.abs() * (0.5 * gamma(r.shape[1]) + 8 * F32), r.dtype)


def residual_norm_back(dr, dy, r, h, gate, post, pre, scale, eps):
    """{name: (value, bound)} of the gradients over rows [N, D], gate [G, D] or None."""
    T, (N, D) = r.dtype, r.shape
    zero = torch.zeros(N, D, dtype=torch.float64, device=r.device)
    dr = zero if dr is None else dr.double()
    rel = 0.5 * gamma(D) + 4 * F32
    out = {}
    e, err = dr, zero
    if pre is not None:
        P, pre64 = pre.dtype, pre.double()
        dy = zero if dy is None else dy.double()
        c = inv_rms(r.double(), eps)
        rhat, p = r.double() * c, dy * pre64
        m = (p * rhat).mean(1, keepdim=True)
        e_m = (gamma(D) + 2 * rel + 4 * F32) * (p * rhat).abs().mean(1, keepdim=True)
        n = c * (p - rhat * m)
        e = dr + n
        err = c * (rhat.abs() * e_m + (p.abs() + (rhat * m).abs()) * (2 * rel + 6 * F32)) + 2 * F32 * (dr.abs() + n.abs())
        dpre = (dy * rhat).sum(0)
        out["dpre"] = (dpre, rounded(dpre, (gamma(N) + rel + 4 * F32) * (dy * rhat).abs().sum(0), P))
    dx = scale * e
    out["dx"] = (dx, rounded(dx, abs(scale) * (err + 2 * F32 * e.abs()), T))
    if h is None:
        return out
    h = h.double()
    a, ra = (1.0, 0.0) if post is None else (inv_rms(h, eps), rel)
    hat = h * a
    g = gate_rows(gate, N) if gate is not None else torch.ones(1, 1, dtype=torch.float64, device=r.device)
    w = 1.0 if post is None else post.double()
    q = e * g * w
    e_q = (g * w).abs() * err + 3 * F32 * q.abs()
    if post is None:
        dh, e_dh = q, e_q
    else:
        m = (q * hat).mean(1, keepdim=True)
        e_m = (e_q * hat.abs()).mean(1, keepdim=True) + (gamma(D) + 2 * ra + 4 * F32) * (q * hat).abs().mean(1, keepdim=True)
        dh = a * (q - hat * m)
        e_dh = a * (e_q + hat.abs() * e_m + (q.abs() + (hat * m).abs()) * (2 * ra + 6 * F32))
        v = e * g * hat
        out["dpost"] = (v.sum(0), rounded(v.sum(0), (gamma(N) + ra + 8 * F32) * v.abs().sum(0) + ((g * hat).abs() * err).sum(0), post.dtype))
    out["dh"] = (dh, rounded(dh, e_dh, T))
    if gate is not None:
        G = gate.shape[0]
        v, e_v = e * hat * w, err * (hat * w).abs()
        fold = lambda t: t.reshape(G, N // G, D).sum(1)
        out["dgate"] = (fold(v), rounded(fold(v), (gamma(N // G) + ra + 8 * F32) * fold(v.abs()) + fold(e_v), gate.dtype))
    return out


def embedding(ids, table, scale, residual=None):
    T, (V, D) = table.dtype, table.shape
    ids = ids.reshape(-1).long()
    inside = (ids >= 0) & (ids < V)
    t = torch.where(inside[:, None], table.double()[ids.clamp(0, V - 1)] * scale, 0.0)
    y = t if residual is None else t + residual.reshape(-1, D).double()
    return y, rounded(y, 2 * F32 * (t.abs() + y.abs()), T)


def embedding_back(dy, ids, rows, scale):
    T, D = dy.dtype, dy.shape[-1]
    ids, dy = ids.reshape(-1).long(), dy.reshape(-1, D).double()
    inside = (ids >= 0) & (ids < rows)
    at = ids[inside]
    zero = torch.zeros(rows, D, dtype=torch.float64, device=dy.device)
    v, size = zero.index_add(0, at, dy[inside]) * scale, zero.index_add(0, at, dy[inside].abs()) * abs(scale)
    n = torch.zeros(rows, dtype=torch.float64, device=dy.device).index_add(0, at, torch.ones(len(at), dtype=torch.float64, device=dy.device))
    return v, rounded(v, gamma(n)[:, None] * size, T)
