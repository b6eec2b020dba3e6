"""The operators of a trained per-pixel (or per-token) decoder block, as calls whose speed and exactness are measured.

A residual gated block, ``x + dropout(ffn(norm(x)))``, sits between the composited feature map and the colour head. Its three
operators have cases here over their whole range, from one row to every pixel of a frame and from a hash grid's 16 feature
channels to rows of thousands:

- ``norm``: layer norm of each row, and its gradients (the weight's and the bias's summed over all rows);
- ``drop``: dropout from a counter-based generator, alone or added to a residual; the backward pass makes the mask again;
- ``ffn``: ``(act(x Wg^T) * (x Wu^T)) Wd^T`` and the gradients of the input and of the three weights.

Each case is one call (``train`` false) or a forward and a backward call (``train`` true). The plain forms are the formulas in
32 bits; the exact ones differentiate the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
_module = None


def _blocks():
    """The framework's module, imported at its first use."""
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nest-splatting_amd"))
        from nest_splat import blocks
        _module = blocks
    return _module


def listed():
    return [
        # The norm of one token's row while answering: nothing but latency.
        dict(name="norm_token", op="norm", dtype="bf16", rows=1, cols=2048, train=False),
        # A training step's norm over every pixel of a 1600 x 1064 frame of 16 levels with 4 features each.
        dict(name="norm_frame", op="norm", dtype="bf16", rows=1600 * 1064, cols=64, train=True),
        # Wide rows in full precision, as a generic model's training step has them.
        dict(name="norm_wide", op="norm", dtype="f32", rows=8192, cols=4096, train=True),
        # A ragged batch: odd counts of rows and columns, so that no row after the first is aligned.
        dict(name="norm_ragged", op="norm", dtype="f16", rows=5003, cols=1155, train=True),
        # Dropout onto the residual over a whole frame, with its backward pass.
        dict(name="drop_frame", op="drop", dtype="bf16", rows=1600 * 1064, cols=64, p=0.1, residual=True, train=True),
        # A small odd batch of a regularised run, forward alone.
        dict(name="drop_ragged", op="drop", dtype="f32", rows=333, cols=1001, p=0.25, residual=False, train=False),
        # One token through a wide block: every weight is read for one row.
        dict(name="ffn_token", op="ffn", dtype="bf16", act="silu", rows=1, cols=2048, hidden=8192, train=False),
        # A small decoding batch: still bound by the weights.
        dict(name="ffn_batch", op="ffn", dtype="f16", act="gelu", rows=32, cols=2048, hidden=8192, train=False),
        # A frame decoded: 1600 x 1064 pixels of 64 features, every one through a narrow block.
        dict(name="ffn_frame", op="ffn", dtype="bf16", act="silu", rows=1600 * 1064, cols=64, hidden=128, train=False),
        # A training step of the narrow block on an 800 x 800 view of 16 levels with 2 features each.
        dict(name="ffn_frame_train", op="ffn", dtype="f16", act="relu", rows=800 * 800, cols=32, hidden=128, train=True),
        # The largest: a training step of a wide block, bound by matrix products.
        dict(name="ffn_wide_train", op="ffn", dtype="bf16", act="silu", rows=8192, cols=2048, hidden=8192, train=True),
        # Odd sizes in full precision, forward and backward.
        dict(name="ffn_ragged_train", op="ffn", dtype="f32", act="gelu", rows=1777, cols=515, hidden=1365, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "drop", "ffn", "ffn"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    train = rng.random() < 0.5
    if op in ("norm", "drop"):
        cols = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(1600 * 1064, (1600 * 1064 * 64 // 2) // cols))
        if op == "norm":
            return dict(op=op, dtype=dtype, rows=rows, cols=cols, train=train)
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, p=round(rng.uniform(0.02, 0.6), 3),
                    residual=rng.random() < 0.5, train=train)
    act = rng.choice(("silu", "gelu", "relu"))
    if rng.random() < 0.5:  # narrow rows, many of them: a frame's pixels
        cols = rng.choice((16, 24, 32, 48, 64, 80, 96, 128, rng.randint(16, 128)))
        hidden = _log_int(rng, 32, 512)
        rows = _log_int(rng, 1024, min(1600 * 1064, (1600 * 1064 * 64 * 128) // (cols * hidden)))
    else:  # wide rows, from one to thousands: a model's tokens
        cols = _log_int(rng, 128, 2048) // 8 * 8 + (rng.randint(1, 7) if rng.random() < 0.25 else 0)
        hidden = _log_int(rng, 256, 8192) // 8 * 8 + (rng.randint(1, 7) if rng.random() < 0.25 else 0)
        rows = _log_int(rng, 1, 8192)
        if dtype == "f32":
            rows = max(1, min(rows, (1 << 33) // (cols * hidden)))
    return dict(op=op, dtype=dtype, act=act, rows=rows, cols=min(cols, 2048), hidden=min(hidden, 8192), train=train)


def prepare(case, seed):
    dev, dt = "cuda", _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    N, D = case["rows"], case["cols"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(scale)

    s = dict(case=case)
    if case["op"] == "norm":
        # features whose channels have means and spreads of their own
        s["x"] = normal(N, D).mul_(normal(D, scale=0.3).abs_().add_(0.3)).add_(normal(D, scale=0.5)).to(dt)
        s["weight"], s["bias"] = normal(D, scale=0.2).add_(1.0).to(dt), normal(D, scale=0.2).to(dt)
    elif case["op"] == "drop":
        s["x"] = normal(N, D).to(dt)
        s["residual"] = normal(N, D).to(dt) if case["residual"] else None
        s["seed"] = (int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) & 0x7FFFFFFFFFFFFFFF
        s["offset"] = int(seed) % 1000
    else:
        H = case["hidden"]
        s["x"] = normal(N, D).to(dt)  # a norm's output
        s["w_gate"] = normal(H, D, scale=math.sqrt(2.0 / (D + H))).to(dt)
        s["w_up"] = normal(H, D, scale=math.sqrt(2.0 / (D + H))).to(dt)
        s["w_down"] = normal(D, H, scale=math.sqrt(2.0 / (D + H))).to(dt)
    if case["train"]:
        s["dy"] = normal(N, D).to(dt)
    return s


def run(state):
    op = state["case"]["op"]
    return (_norm if op == "norm" else _drop if op == "drop" else _ffn)(state)


# ---- layer norm: y = (x - mean) rstd w + b over each row ----

def _norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        B = _blocks()
        y, mean, rstd = B.layer_norm_forward(x, w, b, EPS)
        if not s["case"]["train"]:
            return {"y": y}
        dx, dw, db = B.layer_norm_backward(s["dy"], x, w, mean, rstd)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    x32, w32 = x.float(), w.float()
    c = x32 - x32.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    hat = c * rstd
    y = (hat * w32 + b.float()).to(x.dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dw, db = (dy * hat).sum(0), dy.sum(0)
    g = dy * w32
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": dw.to(w.dtype), "db": db.to(w.dtype)}


# ---- dropout: element i is kept where a 16-bit random number is at least round(p 65536), and scaled by the inverse of the
# share that is kept. Eight elements, 8 c to 8 c + 7, take theirs from one 128-bit block of the ten-round Philox 4x32
# generator (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011), whose counter is
# (c, offset) and whose key is the seed; the low half of a word comes first ----

_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _threshold(p):
    t = int(math.floor(p * 65536.0 + 0.5))
    return t, 65536.0 / (65536 - t) if t < 65536 else 0.0


def _plain_keep(n, t, seed, offset, dev):
    c = torch.arange((n + 7) // 8, device=dev, dtype=torch.int64)
    a, b, d, e = c & _LOW, c >> 32, torch.full_like(c, offset & _LOW), torch.full_like(c, offset >> 32 & _LOW)
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):  # the generator's rounds; a 64-bit product's halves survive the sign
        p0, p1 = a * _M0, d * _M1
        a, b, d, e = (p1 >> 32 & _LOW) ^ b ^ k0, p1 & _LOW, (p0 >> 32 & _LOW) ^ e ^ k1, p0 & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    words = torch.stack((a, b, d, e), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n] >= t


def _drop(s):
    x, p, train = s["x"], s["case"]["p"], s["case"]["train"]
    if own:
        B = _blocks()
        y = B.dropout_forward(x, p, s["seed"], s["offset"], residual=s["residual"])
        return {"y": y, "dx": B.dropout_backward(s["dy"], p, s["seed"], s["offset"])} if train else {"y": y}
    t, scale = _threshold(p)
    keep = _plain_keep(x.numel(), t, s["seed"], s["offset"], x.device).view_as(x)
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        y = s["residual"].float() + y
    out = {"y": y.to(x.dtype)}
    if train:
        out["dx"] = torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)
    return out


# ---- gated feed-forward: h = act(g) u with g = x Wg^T, u = x Wu^T; y = h Wd^T ----

def _act(g, act, slope):
    """act(g), and its slope where it is asked for."""
    if act == "relu":
        on = (g > 0).float()
        return g * on, on
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-g))
        return g * q, q * (1.0 + g * (1.0 - q)) if slope else None
    q = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * q, q + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi)) if slope else None


def _ffn(s):
    x, wg, wu, wd, act, train = s["x"], s["w_gate"], s["w_up"], s["w_down"], s["case"]["act"], s["case"]["train"]
    if own:
        B = _blocks()
        if not train:
            return {"y": B.gated_ffn_forward(x, wg, wu, wd, act)[0]}
        y, kept = B.gated_ffn_forward(x, wg, wu, wd, act, training=True)
        dx, dg, du, dd = B.gated_ffn_backward(s["dy"], x, wg, wu, wd, kept, act)
        return {"y": y, "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    x32, wg32, wu32, wd32 = x.float(), wg.float(), wu.float(), wd.float()
    g, u = x32 @ wg32.T, x32 @ wu32.T
    a, slope = _act(g, act, train)
    h = a * u
    y = (h @ wd32.T).to(x.dtype)
    if not train:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy @ wd32
    dg, du = dh * u * slope, dh * a
    dx = dg @ wg32 + du @ wu32
    return {"y": y, "dx": dx.to(x.dtype), "dw_gate": (dg.T @ x32).to(x.dtype), "dw_up": (du.T @ x32).to(x.dtype),
            "dw_down": (dy.T @ h).to(x.dtype)}


# ---- the definitions in 64 bits ----

def _exact_random16(n, seed, offset, dev):
    """The same numbers from 16-bit limbs: no product here passes 48 bits."""

    def mul(m, v):
        low, high = m * (v & 0xFFFF), m * (v >> 16)
        mid = high + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    blocks = torch.arange((n + 7) // 8, device=dev)
    ctr = [blocks % (1 << 32), blocks // (1 << 32), torch.full_like(blocks, offset % (1 << 32)), torch.full_like(blocks, offset // (1 << 32))]
    key = [seed % (1 << 32), seed // (1 << 32)]
    for r in range(10):
        (h0, l0), (h1, l1) = mul(_M0, ctr[0]), mul(_M1, ctr[2])
        k = [(key[0] + r * _W0) % (1 << 32), (key[1] + r * _W1) % (1 << 32)]
        ctr = [h1 ^ ctr[1] ^ k[0], l1, h0 ^ ctr[3] ^ k[1], l0]
    out = torch.empty((blocks.numel(), 8), dtype=torch.int64, device=dev)
    for j in range(8):
        out[:, j] = (ctr[j // 2] >> (16 * (j % 2))) & 0xFFFF
    return out.view(-1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double().requires_grad_(k not in ("dy", "residual")) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    x = s["x"]
    with torch.enable_grad():
        if case["op"] == "norm":
            named = {"dx": x, "dw": s["weight"], "db": s["bias"]}
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            y = (x - mean) / torch.sqrt(var + EPS) * s["weight"] + s["bias"]
        elif case["op"] == "drop":
            named = {"dx": x}
            t = round(case["p"] * 65536)
            kept = _exact_random16(x.numel(), s["seed"], s["offset"], x.device).view_as(x) >= t
            y = x * (kept.double() * (65536.0 / (65536 - t)))
            y = y if s["residual"] is None else y + s["residual"]
        else:
            named = {"dx": x, "dw_gate": s["w_gate"], "dw_up": s["w_up"], "dw_down": s["w_down"]}
            g = torch.matmul(x, s["w_gate"].t())
            a = torch.clamp(g, min=0) if case["act"] == "relu" else g * torch.sigmoid(g) if case["act"] == "silu" else \
                g * torch.special.ndtr(g)
            y = torch.matmul(a * torch.matmul(x, s["w_up"].t()), s["w_down"].t())
        if not case["train"]:
            return {"y": y.detach()}
        grads = torch.autograd.grad(y, list(named.values()), s["dy"])
    return {"y": y.detach(), **dict(zip(named, grads))}


def work(case):
    N, D, b = case["rows"], case["cols"], _BYTES[case["dtype"]]
    both = 2 if case["train"] else 1
    if case["op"] == "norm":
        return {"bytes": b * both * (2 * N * D + 2 * D), "flops": (8 if both == 1 else 20) * N * D}
    if case["op"] == "drop":
        return {"bytes": b * N * D * (2 * both + int(case["residual"])), "flops": both * N * D}
    H = case["hidden"]
    return {"bytes": b * both * (2 * N * D + 3 * H * D), "flops": 6 * N * D * H * (3 if case["train"] else 1)}
