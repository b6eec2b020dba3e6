"""A trained decoder block and its operators: layer norm, dropout from a
counter-based generator, and a gated feed-forward product, each with its
backward pass, on libnest_splat.

The reference decodes the composited feature map with one small MLP
(hash_encoder/modules.py:551-602) and has none of these; a residual block
x + dropout(ffn(norm(x))) refines the features of every pixel before that MLP
(``GatedRefiner``, ``renderer.HashINGP(refiner=...)``).

Three levels, as elsewhere in this package:

- ``*_forward`` / ``*_backward``: one library call each, on tensors;
- ``layer_norm``, ``dropout``, ``gated_ffn``: the same under autograd;
- ``LayerNorm``, ``Dropout``, ``GatedFFN``, ``GatedRefiner``: modules.

Tensors are on the GPU, of float32, float16 or bfloat16, with any leading
dimensions; sums are float32 and each result is rounded once.  gated_ffn also
rounds what its first products hand to its second ones, h = act(g) u and in
the backward pass dg and du, to the type: in 16 bits its results are off by
about 1.4 times what one rounding makes, and in float16 an h, dg or du past
65504 makes the results that it enters infinite or NaN.  Its float32 products
leave out at most 2^-24 of each (operands below 2^-110 keep their bits down to
2^-133), and a float32 result that an infinity enters may be NaN.  Tensors that are not contiguous are copied first.
Every call is ordered on the current
stream of the tensors' device.  Gradients of gradients are not available.
"""
from __future__ import annotations

import ctypes as ct
import math
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L

_CODE = {torch.float32: L.DTYPE_F32, torch.float16: L.DTYPE_F16, torch.bfloat16: L.DTYPE_BF16}
_NAMED = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_STRUCT_SIZE = ct.sizeof(L.GatedFfn)
_ACT = {"relu": L.ACT_RELU, "silu": L.ACT_SILU, "gelu": L.ACT_GELU}


def _code(t: torch.Tensor, name: str) -> int:
    code = _CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} is {t.dtype}: float32, float16 and bfloat16 are supported")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: the operators run on the GPU")
    return code


def _like(t: torch.Tensor, ref: torch.Tensor, shape, name: str, dtype=None) -> torch.Tensor:
    """t checked against the main tensor's device, a type and a shape, and made contiguous."""
    if t.get_device() != ref.get_device():   # -1 off the GPU; less to build than two devices
        raise ValueError(f"{name} is on {t.device}, expected {ref.device}")
    if t.dtype is not (dtype or ref.dtype):
        raise TypeError(f"{name} is {t.dtype}, expected {dtype or ref.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() else t.detach().contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t at an address of a multiple of 16 bytes: a view into the middle of another tensor is copied."""
    return t.clone() if t.data_ptr() % 16 else t


# the current stream and device without the objects around them, where this torch has them
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name: str, device: torch.device, *args) -> None:
    """Calls a library function on the device's current stream, with the device current."""
    function = getattr(L.lib(), name)
    index = device.index
    if index == _raw_device():
        rc = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = function(*args, _raw_stream(index))
    if rc != L.NEST_OK:
        L.check(rc, name)


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _whole(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.detach().contiguous()


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---- layer norm ----

def _norm_args(x, weight, bias, eps):
    code = _code(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs a last dimension of at least 1")
    D = x.shape[-1]
    pdt = weight.dtype
    if pdt not in (torch.float32, x.dtype):
        raise TypeError(f"weight is {pdt}: float32 or the type of x ({x.dtype}) is expected")
    weight = _like(weight, x, (D,), "weight", pdt)
    if bias is not None:
        bias = _like(bias, x, (D,), "bias", pdt)
    if eps is not None and not eps >= 0:
        raise ValueError("eps must not be negative")
    return code, _CODE[pdt], _whole(x), weight, bias, x.numel() // D, D


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last dimension; mean and rstd are float32 [rows]."""
    code, pcode, x, weight, bias, rows, D = _norm_args(x, weight, bias, eps)
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    _call("nest_layer_norm", x.device, rows, D, code, pcode, _at(x), _at(weight), _at(bias), eps, _at(y), _at(mean), _at(rstd))
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, with_bias: bool = True):
    """(dx, dweight, dbias) from dy and what layer_norm_forward returned; dbias is None without ``with_bias``."""
    code, pcode, x, weight, _, rows, D = _norm_args(x, weight, None, None)
    dy = _like(dy, x, x.shape, "dy")
    mean, rstd = (_like(t, x, (rows,), n, torch.float32) for t, n in ((mean, "mean"), (rstd, "rstd")))
    dx, dw = torch.empty_like(x), torch.empty_like(weight)
    db = torch.empty_like(weight) if with_bias else None
    nbytes = L.lib().nest_layer_norm_backward_workspace_size(rows, D, code)
    ws = _workspace(nbytes, x.device)
    _call("nest_layer_norm_backward", x.device, rows, D, code, pcode, _at(dy), _at(x), _at(weight), _at(mean), _at(rstd), _at(dx),
          _at(dw), _at(db), _at(ws), nbytes)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.with_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*layer_norm_backward(dy, *ctx.saved_tensors, with_bias=ctx.with_bias), None)


def layer_norm(x, weight, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """layer_norm_forward's y under autograd (x, weight and bias)."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---- dropout ----

def dropout_forward(x: torch.Tensor, p: float, seed: int, offset: int = 0,
                    residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x where it is kept, scaled by the inverse of the share that is kept, else 0; plus ``residual``.

    The mask is a function of p, seed, offset (64-bit numbers) and an element's place in x alone, so the same call
    repeats it; take another offset for each use. p acts in steps of 1/65536. A HIP graph records seed and offset as
    they were."""
    code = _code(x, "x")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("seed and offset are unsigned 64-bit numbers")
    if residual is not None:
        residual = _like(residual, x, x.shape, "residual")
    x = _whole(x)
    y = torch.empty_like(x)
    _call("nest_dropout", x.device, x.numel(), code, _at(x), _at(residual), p, seed, offset, _at(y))
    return y


def dropout_backward(dy: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """The gradient of x from dy, with the mask made again; the residual's gradient is dy itself."""
    return dropout_forward(dy, p, seed, offset)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, residual):
        ctx.args = (p, seed, offset)
        return dropout_forward(x, p, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = dropout_backward(dy, *ctx.args) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def dropout(x, p: float, seed: int, offset: int = 0, residual=None) -> torch.Tensor:
    """dropout_forward under autograd (x and residual)."""
    return _Dropout.apply(x, p, seed, offset, residual)


# ---- gated feed-forward ----

def _weight(t, ref, shape, name):
    return _aligned(_like(t, ref, shape, name))


def _gated(x, w_gate, w_up, w_down, activation):
    code = _code(x, "x")
    act = _ACT.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_ACT)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError("x needs a last dimension, the weights are [out, in] matrices")
    I, (H, _), (O, _) = x.shape[-1], w_gate.shape, w_down.shape
    if I < 1 or H < 1 or O < 1:
        raise ValueError("in_features, hidden and out_features must be at least 1")
    x = _aligned(_whole(x))
    up = (H, I)
    w_gate, w_up, w_down = _weight(w_gate, x, up, "w_gate"), _weight(w_up, x, up, "w_up"), _weight(w_down, x, (O, H), "w_down")
    f = L.GatedFfn(_STRUCT_SIZE, code, act, I, H, O, x.numel() // I, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr())
    return f, x, (w_gate, w_up, w_down)


def _gated_sizes(f):
    """Bytes of (kept, a forward's workspace, a backward's with kept, without)."""
    kept, fwd, bwd, alone = ct.c_size_t(), ct.c_size_t(), ct.c_size_t(), ct.c_size_t()
    rc = L.lib().nest_gated_ffn_sizes(f, kept, fwd, bwd, alone)
    if rc != L.NEST_OK:
        L.check(rc, "nest_gated_ffn_sizes")
    return kept.value, fwd.value, bwd.value, alone.value


def gated_ffn_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                      activation: str = "silu", training: bool = False):
    """(y, kept): y = (act(x w_gate^T) * (x w_up^T)) w_down^T for x [..., in], w_gate and w_up [hidden, in], w_down
    [out, hidden], all of one type. ``training``: kept is what gated_ffn_backward takes to save work (it may be None,
    where computing it again costs less); it is None otherwise."""
    f, x, ws = _gated(x, w_gate, w_up, w_down, activation)
    kept_bytes, fwd_bytes, _, _ = _gated_sizes(f)
    O = f.out_features
    y = torch.empty_like(x) if O == x.shape[-1] else torch.empty(x.shape[:-1] + (O,), dtype=x.dtype, device=x.device)
    kept = _workspace(kept_bytes, x.device) if training else None
    work = _workspace(fwd_bytes, x.device)
    _call("nest_gated_ffn_forward", x.device, f, _at(y), _at(kept), _at(work), fwd_bytes)
    return y, kept


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                       w_down: torch.Tensor, kept: Optional[torch.Tensor] = None, activation: str = "silu",
                       needs=(True, True, True, True)):
    """(dx, dw_gate, dw_up, dw_down); ``needs``: which of them are wanted, the others are None. ``kept``: what the
    forward call with the same arguments returned; None computes it again."""
    f, x, ws = _gated(x, w_gate, w_up, w_down, activation)
    dy = _aligned(_like(dy, x, x.shape[:-1] + (f.out_features,), "dy"))
    kept_bytes, _, bwd_bytes, alone_bytes = _gated_sizes(f)
    if kept is not None and (kept.dtype != torch.uint8 or kept.numel() != kept_bytes or not kept.is_contiguous()
                             or kept.device != x.device):
        raise ValueError("kept is not what gated_ffn_forward(training=True) returned for these arguments")
    grads = [torch.empty_like(t) if n else None for t, n in zip((x, *ws), needs)]
    nbytes = bwd_bytes if kept is not None else alone_bytes
    work = _workspace(nbytes, x.device)
    _call("nest_gated_ffn_backward", x.device, f, _at(dy), _at(kept), *(_at(g) for g in grads), _at(work), nbytes)
    return tuple(grads)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, recording):
        # needs_input_grad is that of the tensors, whether or not gradients are recorded
        y, kept = gated_ffn_forward(x, w_gate, w_up, w_down, activation, training=recording and any(ctx.needs_input_grad))
        ctx.save_for_backward(x, w_gate, w_up, w_down, kept)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        grads = gated_ffn_backward(dy, *ctx.saved_tensors, ctx.activation, ctx.needs_input_grad[:4])
        return (*grads, None, None)


def gated_ffn(x, w_gate, w_up, w_down, activation: str = "silu") -> torch.Tensor:
    """gated_ffn_forward's y under autograd (x and the three weights)."""
    return _GatedFfn.apply(x, w_gate, w_up, w_down, activation, torch.is_grad_enabled())


# ---- modules ----

class LayerNorm(nn.Module):
    """layer_norm over the last dimension with float32 weight and bias, for rows of any of the types."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(features))
        self.bias = nn.Parameter(torch.zeros(features)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)


# the backward pass that this call is made from, -1 outside of any
_backward_id = getattr(torch._C, "_current_graph_task_id", lambda: -1)


class Dropout(nn.Module):
    """dropout while training, with a new mask each call. In evaluation x passes through (plus the residual).

    Without ``seed`` each call draws its key from torch's CPU generator: torch.manual_seed governs the masks, modules and
    differently seeded ranks have masks of their own, and a forward that torch.utils.checkpoint recomputes, with the
    generator's state restored, draws its mask again. With ``seed`` the module counts its calls under that key, and its
    state dict keeps the count, so a resumed run draws the masks that follow; such a count cannot be taken back for a
    recomputed forward, and replicas would count on copies: both raise."""

    def __init__(self, p: float = 0.1, seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        self.p, self.seed, self.offset = float(p), None if seed is None else int(seed), 0

    def get_extra_state(self):
        return {"seed": self.seed, "offset": self.offset}

    def set_extra_state(self, state):
        self.seed, self.offset = state["seed"], state["offset"]

    def _key(self):
        """(seed, offset) of this call."""
        if self.seed is None:
            return int(torch.empty((), dtype=torch.int64, device="cpu").random_()), 0
        if _backward_id() != -1:
            raise RuntimeError("a recomputed forward would draw another mask from a Dropout with a seed of its own: leave seed "
                               "out (torch's generator then repeats the mask), or call dropout with an offset")
        if getattr(self, "_is_replica", False):
            raise RuntimeError("a replica of a Dropout with a seed of its own would repeat its masks each step: leave seed out")
        self.offset += 1
        return self.seed, self.offset - 1

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return dropout(x, self.p, *self._key(), residual)


class GatedFFN(nn.Module):
    """gated_ffn with float32 weights, computed in ``dtype`` (x and the weights are cast to it, y has it)."""

    def __init__(self, features: int, hidden: int, out_features: Optional[int] = None, activation: str = "silu", dtype="bf16",
                 seed: int = 0):
        super().__init__()
        if activation not in _ACT:
            raise ValueError(f"activation must be one of {sorted(_ACT)}, got {activation!r}")
        self.activation = activation
        self.dtype = _NAMED.get(dtype, dtype)
        if self.dtype not in _CODE:
            raise TypeError(f"dtype {dtype!r}: float32, float16 and bfloat16 are supported")
        g = torch.Generator().manual_seed(seed)

        def xavier(o, i):
            return nn.Parameter((torch.rand((o, i), generator=g) * 2 - 1) * math.sqrt(6.0 / (i + o)))
        self.w_gate, self.w_up = xavier(hidden, features), xavier(hidden, features)
        self.w_down = xavier(features if out_features is None else out_features, hidden)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        t = self.dtype
        return gated_ffn(x.to(t), self.w_gate.to(t), self.w_up.to(t), self.w_down.to(t), self.activation)


class GatedRefiner(nn.Module):
    """``depth`` residual blocks x + dropout(ffn(norm(x))) over the feature channels of every pixel.

    The rows run through the blocks in ``dtype``. The down projections start at zero, so a new refiner returns its input
    rounded to dtype; with the colour MLP's own 16-bit type that leaves the decoded image as it was, since the MLP
    rounds its features to that type. ``seed`` makes the weights; the masks come from torch's generator (see Dropout)."""

    def __init__(self, features: int, hidden: Optional[int] = None, depth: int = 1, p: float = 0.1, activation: str = "silu",
                 dtype="bf16", seed: int = 0):
        super().__init__()
        self.features = int(features)
        self.dtype = _NAMED.get(dtype, dtype)
        self.norms = nn.ModuleList(LayerNorm(features) for _ in range(depth))
        self.ffns = nn.ModuleList(GatedFFN(features, hidden or 2 * features, None, activation, dtype, seed + k) for k in range(depth))
        self.drops = nn.ModuleList(Dropout(p) for _ in range(depth))
        for f in self.ffns:
            nn.init.zeros_(f.w_down)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., features] of any of the types -> the same shape and type."""
        if x.shape[-1] != self.features:
            raise ValueError(f"expected {self.features} feature channels, got {x.shape[-1]}")
        y = x.to(self.dtype)
        for norm, ffn, drop in zip(self.norms, self.ffns, self.drops):
            y = drop(ffn(norm(y)), residual=y)
        return y.to(x.dtype)

    def refine_image(self, color: torch.Tensor) -> torch.Tensor:
        """A feature map [C, H, W] refined pixel by pixel."""
        C, H, W = color.shape
        return self(color.reshape(C, -1).t()).t().reshape(C, H, W).contiguous()
