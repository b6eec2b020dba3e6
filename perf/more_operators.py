"""The operators of a residual block that is conditioned on the view (or the token), as calls whose speed and exactness are measured.

A refiner between the composited feature map and the colour head adds an embedding of the view to each pixel's features and runs
them through dense layers, each branch joined to the residual stream between two norms. Its four operators have cases here over
their whole range, from one row to every pixel of a frame and from a hash grid's 16 feature channels to rows of thousands:

- ``linear``: ``act(x W^T + b) + residual`` and its gradients;
- ``saved``: the same training step with what its backward pass needs kept in 8 bits; with ``pack`` alone, rows to 8 bits and back;
- ``rnorm``: ``t = h / rms(h) * post``, ``r = scale x + gate t``, ``y = r / rms(r) * pre`` (``r`` as it is stored), and its gradients;
- ``embed``: ``residual + scale table[id]`` (nothing for an id outside the table), and the gradient of the table.

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
EPS = 1e-6
FRAME = 1600 * 1064
_module = None


def _ops():
    """The framework's module, imported at its first use."""
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nest-splatting_amd"))
        from nest_splat import residual
        _module = residual
    return _module


def listed():
    return [
        # One token through a wide layer while answering: every weight is read for one row.
        dict(name="linear_token", op="linear", dtype="bf16", act="silu", rows=1, cols=2048, out=8192, residual=False, train=False),
        # A training step of a narrow layer on every pixel of a 1600 x 1064 frame of 16 levels with 4 features each.
        dict(name="linear_frame_train", op="linear", dtype="bf16", act="gelu", rows=FRAME, cols=64, out=64, residual=True, train=True),
        # The largest: a training step of a wide layer, bound by matrix products.
        dict(name="linear_wide_train", op="linear", dtype="bf16", act="gelu", rows=8192, cols=2048, out=8192, residual=False, train=True),
        # Odd sizes in full precision.
        dict(name="linear_ragged_train", op="linear", dtype="f32", act="silu", rows=1777, cols=515, out=1365, residual=True, train=True),
        # A frame's features to 8 bits and back, as a checkpoint holds them.
        dict(name="pack_frame", op="pack", dtype="bf16", rows=FRAME, cols=64),
        # A narrow layer on an 800 x 800 view of 16 levels with 2 features each, trained from 8 bits.
        dict(name="saved_frame_train", op="saved", dtype="f16", act="relu", rows=800 * 800, cols=32, out=128),
        # A wide layer trained from 8 bits.
        dict(name="saved_wide_train", op="saved", dtype="bf16", act="silu", rows=8192, cols=2048, out=2048),
        # One token's branch joined to its residual stream and normed for the next block: nothing but latency.
        dict(name="rnorm_token", op="rnorm", dtype="bf16", rows=1, cols=2048, gates=1, scale=1.0, train=False),
        # A training step's join over every pixel of a frame, gated by channel.
        dict(name="rnorm_frame_train", op="rnorm", dtype="bf16", rows=FRAME, cols=64, gates=1, scale=1.0, train=True),
        # Wide rows in full precision, a gate for each of eight sequences.
        dict(name="rnorm_wide_train", op="rnorm", dtype="f32", rows=8192, cols=4096, gates=8, scale=0.7, train=True),
        # An embedding of each of 300 views added to a frame's worth of pixels drawn from them, with its gradient.
        dict(name="embed_views_train", op="embed", dtype="bf16", rows=FRAME, cols=64, table=300, residual=True, skew=0.0, train=True),
        # A batch of tokens from a vocabulary, few of them frequent, and the whole table's gradient.
        dict(name="embed_tokens_train", op="embed", dtype="bf16", rows=8192, cols=2048, table=32000, residual=False, skew=3.0, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "saved", "pack", "rnorm", "rnorm", "embed", "embed"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    train = rng.random() < 0.5
    if op in ("linear", "saved"):
        act = rng.choice(("none", "relu", "silu", "gelu"))
        if act == "relu" and dtype == "f32":  # whose slope turns on the order of a sum that is nearly zero
            act = "silu"
        if rng.random() < 0.5:  # narrow rows, many of them: a frame's pixels
            cols = rng.choice((16, 24, 32, 48, 64, 96, 128, rng.randint(16, 128)))
            out = rng.choice((16, 32, 64, 128, rng.randint(16, 128)))
            rows = _log_int(rng, 1024, min(FRAME, FRAME * 64 // max(cols, out)))
        else:  # wide rows, from one to thousands: a model's tokens
            cols = _log_int(rng, 128, 2048) // 8 * 8 + (rng.randint(1, 7) if rng.random() < 0.25 else 0)
            out = _log_int(rng, 128, 8192) // 8 * 8 + (rng.randint(1, 7) if rng.random() < 0.25 else 0)
            rows = _log_int(rng, 1, 8192)
            cols, out = min(cols, 2048), min(out, 8192)
            if dtype == "f32":
                rows = max(1, min(rows, (1 << 34) // (cols * out)))
        if op == "saved":
            return dict(op=op, dtype=dtype, act=act, rows=rows, cols=cols, out=out)
        return dict(op=op, dtype=dtype, act=act, rows=rows, cols=cols, out=out, residual=rng.random() < 0.5, train=train)
    cols = _log_int(rng, 16, 8192)
    rows = _log_int(rng, 1, min(FRAME, FRAME * 32 // cols))
    if op == "pack":
        return dict(op=op, dtype=dtype, rows=rows, cols=cols)
    if op == "rnorm":
        gates = rng.choice((0, 1, 1, rng.choice((2, 4, 8)), rows))
        gates = 1 if gates == rows and rows * cols > 1 << 25 else gates
        if gates > 1:
            rows = max(1, rows // gates) * gates
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, gates=gates, scale=rng.choice((1.0, round(rng.uniform(0.3, 1.0), 3))), train=train)
    table = _log_int(rng, 2, max(2, min(100000, (1 << 26) // cols)))
    return dict(op=op, dtype=dtype, rows=rows, cols=cols, table=table, residual=rng.random() < 0.5, skew=rng.choice((0.0, 2.0, 4.0)),
                train=train)


def prepare(case, seed):
    dev, dt = "cuda", _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    N, D = case["rows"], case["cols"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(scale)

    def features(rows, cols):  # channels with means and spreads of their own
        return normal(rows, cols).mul_(normal(cols, scale=0.3).abs_().add_(0.3)).add_(normal(cols, scale=0.3))

    s = dict(case=case)
    op = case["op"]
    if op in ("linear", "saved"):
        H = case["out"]
        s["x"] = normal(N, D).to(dt)  # a norm's output
        s["weight"] = normal(H, D, scale=math.sqrt(1.0 / D)).to(dt)
        s["bias"] = normal(H, scale=0.2).to(dt)
        s["residual"] = normal(N, H).to(dt) if case.get("residual") else None
        if case.get("train", True):
            s["dy"] = normal(N, H).to(dt)
    elif op == "pack":
        s["x"] = features(N, D).to(dt)
    elif op == "rnorm":
        s["x"], s["h"] = features(N, D).to(dt), normal(N, D, scale=2.0).to(dt)
        s["post"], s["pre"] = normal(D, scale=0.2).add_(1.0).to(dt), normal(D, scale=0.2).add_(1.0).to(dt)
        s["gate"] = normal(case["gates"], D, scale=0.3).add_(0.5).to(dt) if case["gates"] else None
        if case["train"]:
            s["dr"], s["dy"] = normal(N, D).to(dt), normal(N, D).to(dt)
    else:
        V = case["table"]
        u = torch.rand(N, generator=g, device=dev)  # skew: low ids are the frequent ones
        ids = (u.pow_(1.0 + case["skew"]) * V).long().clamp_(max=V - 1)
        s["ids"] = torch.where(torch.rand(N, generator=g, device=dev) < 0.02, -1, ids)  # some rows belong to no view
        s["table"] = normal(V, D, scale=0.5).to(dt)
        s["residual"] = features(N, D).to(dt) if case["residual"] else None
        s["scale"] = 1.25
        if case["train"]:
            s["dy"] = normal(N, D).to(dt)
    return s


def run(state):
    return {"linear": _linear, "saved": _saved, "pack": _pack, "rnorm": _rnorm, "embed": _embed}[state["case"]["op"]](state)


# ---- linear: y = act(z) + residual with z = x W^T + b ----

def _act(z, act, slope):
    """act(z), and its slope where it is asked for."""
    if act == "none":
        return z, torch.ones_like(z) if slope else None
    if act == "relu":
        on = (z > 0).float()
        return z * on, on
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-z))
        return z * q, q * (1.0 + z * (1.0 - q)) if slope else None
    q = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * q, q + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)) if slope else None


def _name(act):
    return None if act == "none" else act


def _linear(s):
    x, w, b, r, act, train = s["x"], s["weight"], s["bias"], s["residual"], s["case"]["act"], s["case"]["train"]
    if own:
        R = _ops()
        y, kept = R.linear_forward(x, w, b, _name(act), r, training=train)
        if not train:
            return {"y": y}
        dx, dw, db = R.linear_backward(s["dy"], x, w, kept, _name(act))
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    x32, w32 = x.float(), w.float()
    a, slope = _act(x32 @ w32.T + b.float(), act, train)
    y = (a if r is None else a + r.float()).to(x.dtype)
    if not train:
        return {"y": y}
    dz = s["dy"].float() * slope
    return {"y": y, "dx": (dz @ w32).to(x.dtype), "dw": (dz.T @ x32).to(x.dtype), "db": dz.sum(0).to(x.dtype)}


# ---- kept in 8 bits: 32 values of a row share a step of 2^(floor(log2 of the largest) - 6) and are held as whole numbers of
# it, -127 to 127; an activation's slope is held in steps of 1/200 (of float32 rows, whose other operands deserve more: 1/26000) ----

def _steps(case):
    return 26000.0 if case["dtype"] == "f32" and case["act"] in ("silu", "gelu") else 200.0


def _plain_pack(x):
    """What the 8 bits of x stand for, in float32."""
    N, D = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -D % 32)).view(N, -1, 32)
    most = v.abs().amax(2, keepdim=True)
    e = (most.view(torch.int32) >> 23).clamp(min=1) - 127           # floor(log2), -126 below the normal numbers
    up = ((133 - e).clamp(max=254) << 23).view(torch.float32)        # 2^(6 - e)
    down = ((121 + e).clamp(min=1) << 23).view(torch.float32)
    return ((v * up).round().clamp(-127, 127) * down).view(N, -1)[:, :D]


def _saved(s):
    x, w, b, dy, act = s["x"], s["weight"], s["bias"], s["dy"], s["case"]["act"]
    if own:
        R = _ops()
        y, kept = R.linear_forward(x, w, b, _name(act), training=True, save8=True)
        dx, dw, db = R.linear_backward(dy, R.pack8(x), w, kept, _name(act))
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    x32, w32 = x.float(), w.float()
    a, slope = _act(x32 @ w32.T + b.float(), act, True)
    dz = dy.float() * (torch.round(slope * _steps(s["case"])) / _steps(s["case"]))
    return {"y": a.to(x.dtype), "dx": (dz @ w32).to(x.dtype), "dw": (dz.T @ _plain_pack(x)).to(x.dtype), "db": dz.sum(0).to(x.dtype)}


def _pack(s):
    if own:
        R = _ops()
        return {"x": R.unpack8(R.pack8(s["x"]))}
    return {"x": _plain_pack(s["x"]).to(s["x"].dtype)}


# ---- the residual stream between two root-mean-square norms ----

def _rnorm(s):
    x, h, gate, post, pre, case = s["x"], s["h"], s["gate"], s["post"], s["pre"], s["case"]
    if own:
        R = _ops()
        r, y, stats = R.residual_norm_forward(x, h, gate, post, pre, case["scale"], EPS)
        if not case["train"]:
            return {"r": r, "y": y}
        dx, dh, dgate, dpost, dpre = R.residual_norm_backward(s["dr"], s["dy"], r, h, gate, post, pre, stats, case["scale"])
        out = {"r": r, "y": y, "dx": dx, "dh": dh, "dpost": dpost, "dpre": dpre}
        return out if gate is None else {**out, "dgate": dgate}
    T, D, scale, G = x.dtype, x.shape[1], case["scale"], max(case["gates"], 1)
    x32, h32, post32, pre32 = x.float(), h.float(), post.float(), pre.float()
    a = torch.rsqrt((h32 * h32).mean(1, keepdim=True) + EPS)
    hat = h32 * a
    t = hat * post32
    gated = t if gate is None else (t.view(G, -1, D) * gate.float()[:, None]).view(-1, D)
    r = (scale * x32 + gated).to(T)
    r32 = r.float()
    c = torch.rsqrt((r32 * r32).mean(1, keepdim=True) + EPS)
    rhat = r32 * c
    y = (rhat * pre32).to(T)
    if not case["train"]:
        return {"r": r, "y": y}
    dy = s["dy"].float()
    p = dy * pre32
    dr = s["dr"].float() + c * (p - rhat * (p * rhat).mean(1, keepdim=True))
    out = {"r": r, "y": y, "dx": (scale * dr).to(T)}
    dt = dr if gate is None else (dr.view(G, -1, D) * gate.float()[:, None]).view(-1, D)
    q = dt * post32
    out["dh"] = (a * (q - hat * (q * hat).mean(1, keepdim=True))).to(T)
    out["dpost"], out["dpre"] = (dt * hat).sum(0).to(T), (dy * rhat).sum(0).to(T)
    return out if gate is None else {**out, "dgate": (dr * t).view(G, -1, D).sum(1).to(T)}


# ---- embedding ----

def _embed(s):
    ids, table, r, scale, case = s["ids"], s["table"], s["residual"], s["scale"], s["case"]
    if own:
        R = _ops()
        y = R.embedding_forward(ids, table, scale, r)
        return {"y": y, "dtable": R.embedding_backward(s["dy"], ids, table.shape[0], scale)} if case["train"] else {"y": y}
    inside = ((ids >= 0) & (ids < table.shape[0]))[:, None]
    at = ids.clamp(0, table.shape[0] - 1)
    y = torch.where(inside, table.float()[at] * scale, 0.0)
    y = (y if r is None else r.float() + y).to(table.dtype)
    if not case["train"]:
        return {"y": y}
    d = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    d.index_add_(0, at, torch.where(inside, s["dy"].float(), 0.0))
    return {"y": y, "dtable": (d * scale).to(table.dtype)}


# ---- the definitions in 64 bits ----

def _exact_act(z, act):
    if act == "none":
        return z
    return torch.clamp(z, min=0) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z * torch.special.ndtr(z)


def _exact_pack(x):
    """Group by group: the largest over its own fraction of a power of two, the nearest whole numbers of the step."""
    N, D = x.shape
    out = torch.empty_like(x)
    for c in range(0, D, 32):
        v = x[:, c:c + 32]
        most = v.abs().max(1, keepdim=True).values
        step = torch.where(most > 0, most / torch.frexp(most)[0] / 128, 1.0)   # a power of two: the division is exact
        out[:, c:c + 32] = torch.clamp(torch.round(v / step), -127.0, 127.0) * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    T = _DTYPES[case["dtype"]]
    leaves = ("x", "weight", "bias", "h", "gate", "post", "pre", "table")
    s = {k: v.double().requires_grad_(k in leaves) if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    op = case["op"]
    if op == "pack":
        return {"x": _exact_pack(s["x"].detach())}
    with torch.enable_grad():
        if op in ("linear", "saved"):
            z = torch.nn.functional.linear(s["x"], s["weight"], s["bias"])
            y = _exact_act(z, case["act"])
            if op == "saved":
                slope = torch.ones_like(z) if case["act"] == "none" else torch.autograd.grad(y, z, torch.ones_like(z), retain_graph=True)[0]
                with torch.no_grad():
                    dz = s["dy"] * torch.round(slope * _steps(case)) / _steps(case)
                    return {"y": y.detach(), "dx": torch.matmul(dz, s["weight"]), "dw": torch.matmul(dz.t(), _exact_pack(s["x"].detach())),
                            "db": dz.sum(0)}
            if s["residual"] is not None:
                y = y + s["residual"]
            outs, grads_of, named = {"y": y}, (s["dy"],) if case["train"] else (), {"dx": s["x"], "dw": s["weight"], "db": s["bias"]}
        elif op == "rnorm":
            N, D, G = case["rows"], case["cols"], max(case["gates"], 1)

            def rms_normed(v):
                return v / torch.sqrt(v.square().sum(-1, keepdim=True) / D + EPS)

            t = rms_normed(s["h"]) * s["post"]
            if s["gate"] is not None:
                t = t * s["gate"].repeat_interleave(N // G, 0)
            r = s["x"] * case["scale"] + t
            r = r + (r.detach().to(T).double() - r.detach())   # the norm before the next block is that of the stored stream
            y = rms_normed(r) * s["pre"]
            outs, grads_of = {"r": r, "y": y}, (s["dr"], s["dy"]) if case["train"] else ()
            named = {"dx": s["x"], "dh": s["h"], "dpost": s["post"], "dpre": s["pre"]}
            if s["gate"] is not None:
                named["dgate"] = s["gate"]
        else:
            V = case["table"]
            rows = torch.cat((s["table"], s["table"].new_zeros(1, case["cols"])))  # the last row: of no id
            at = torch.where((s["ids"] < 0) | (s["ids"] >= V), V, s["ids"])
            y = rows.index_select(0, at) * s["scale"]
            if s["residual"] is not None:
                y = y + s["residual"]
            outs, grads_of, named = {"y": y}, (s["dy"],) if case["train"] else (), {"dtable": s["table"]}
        if not case["train"]:
            return {k: v.detach() for k, v in outs.items()}
        grads = torch.autograd.grad(list(outs.values()), list(named.values()), grads_of)
    return {**{k: v.detach() for k, v in outs.items()}, **dict(zip(named, grads))}


def work(case):
    N, D, b, op = case["rows"], case["cols"], _BYTES[case["dtype"]], case["op"]
    train = case.get("train", True)
    if op in ("linear", "saved"):
        H = case["out"]
        arrays = N * D + D * H + H + N * H * (1 + int(bool(case.get("residual"))))      # x, weight, bias, y, residual
        if train:
            arrays += N * H + N * D + D * H + H                                         # dy, and the gradients
        return {"bytes": b * arrays, "flops": 2 * N * D * H * (3 if train else 1)}
    if op == "pack":
        return {"bytes": 2 * b * N * D, "flops": 4 * N * D}
    if op == "rnorm":
        arrays = 4 * N * D + 2 * D + case["gates"] * D                                  # x, h, r, y
        if train:
            arrays += 4 * N * D + 2 * D + case["gates"] * D                             # dr, dy, dx, dh
        return {"bytes": b * arrays, "flops": (30 if train else 9) * N * D}
    V = case["table"]
    arrays = N * D * (1 + int(case["residual"])) + min(N, V) * D
    if train:
        arrays += N * D + V * D
    return {"bytes": b * arrays + 8 * N, "flops": (4 if train else 2) * N * D}
