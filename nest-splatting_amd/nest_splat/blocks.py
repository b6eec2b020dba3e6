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
dimensions; sums are float32 and each result is rounded once.  Tensors that
are not contiguous are copied first.  Every call is ordered on the current
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
    if t.device != ref.device:
        raise ValueError(f"{name} is on {t.device}, expected {ref.device}")
    if t.dtype != (dtype or ref.dtype):
        raise TypeError(f"{name} is {t.dtype}, expected {dtype or ref.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.detach().contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t at an address of a multiple of 16 bytes: a view into the middle of another tensor is copied."""
    return t.clone() if t.data_ptr() % 16 else t


class _on:
    """Makes the tensors' device the current one around a launch, where it is not already."""

    def __init__(self, device: torch.device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


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
    return code, _CODE[pdt], x.detach().contiguous(), weight, bias, x.numel() // D, D


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last dimension; mean and rstd are float32 [rows]."""
    code, pcode, x, weight, bias, rows, D = _norm_args(x, weight, bias, eps)
    y = torch.empty_like(x)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    with _on(x.device):
        L.check(L.lib().nest_layer_norm(rows, D, code, pcode, L.ptr(x), L.ptr(weight), L.ptr(bias), float(eps),
                                        L.ptr(y), L.ptr(stats[0]), L.ptr(stats[1]), L.stream_ptr(x.device)),
                "nest_layer_norm")
    return y, stats[0], stats[1]


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, with_bias: bool = True):
    """(dx, dweight, dbias) from dy and what layer_norm_forward returned; dbias is None without ``with_bias``."""
    code, pcode, x, weight, _, rows, D = _norm_args(x, weight, None, None)
    dy = _like(dy, x, x.shape, "dy")
    mean, rstd = (_like(t, x, (rows,), n, torch.float32) for t, n in ((mean, "mean"), (rstd, "rstd")))
    dx, dw = torch.empty_like(x), torch.empty_like(weight)
    db = torch.empty_like(weight) if with_bias else None
    lib = L.lib()
    nbytes = lib.nest_layer_norm_backward_workspace_size(rows, D, code)
    ws = _workspace(nbytes, x.device)
    with _on(x.device):
        L.check(lib.nest_layer_norm_backward(rows, D, code, pcode, L.ptr(dy), L.ptr(x), L.ptr(weight), L.ptr(mean),
                                             L.ptr(rstd), L.ptr(dx), L.ptr(dw), L.ptr(db), L.ptr(ws), nbytes,
                                             L.stream_ptr(x.device)), "nest_layer_norm_backward")
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
    x = x.detach().contiguous()
    y = torch.empty_like(x)
    with _on(x.device):
        L.check(L.lib().nest_dropout(x.numel(), code, L.ptr(x), L.ptr(residual), float(p), seed, offset, L.ptr(y),
                                     L.stream_ptr(x.device)), "nest_dropout")
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

def _gated(x, w_gate, w_up, w_down, activation):
    code = _code(x, "x")
    if activation not in _ACT:
        raise ValueError(f"activation must be one of {sorted(_ACT)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError("x needs a last dimension, the weights are [out, in] matrices")
    I, H, O = x.shape[-1], w_gate.shape[0], w_down.shape[0]
    if min(I, H, O) < 1:
        raise ValueError("in_features, hidden and out_features must be at least 1")
    x = _aligned(x.detach().contiguous())
    ws = tuple(_aligned(_like(w, x, s, n)) for w, s, n in ((w_gate, (H, I), "w_gate"), (w_up, (H, I), "w_up"), (w_down, (O, H), "w_down")))
    rows = x.numel() // I
    f = L.GatedFfn(ct.sizeof(L.GatedFfn), code, _ACT[activation], I, H, O, rows, x.data_ptr(), *(w.data_ptr() for w in ws))
    return f, x, ws


def _gated_sizes(f):
    s = [ct.c_size_t() for _ in range(4)]
    L.check(L.lib().nest_gated_ffn_sizes(ct.byref(f), *(ct.byref(v) for v in s)), "nest_gated_ffn_sizes")
    return [v.value for v in s]


def gated_ffn_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                      activation: str = "silu", training: bool = False):
    """(y, kept): y = (act(x w_gate^T) * (x w_up^T)) w_down^T for x [..., in], w_gate and w_up [hidden, in], w_down
    [out, hidden], all of one type. ``training``: kept is what gated_ffn_backward takes to save work (it may be None,
    where computing it again costs less); it is None otherwise."""
    f, x, ws = _gated(x, w_gate, w_up, w_down, activation)
    kept_bytes, fwd_bytes, _, _ = _gated_sizes(f)
    y = torch.empty(x.shape[:-1] + (f.out_features,), dtype=x.dtype, device=x.device)
    kept = _workspace(kept_bytes, x.device) if training else None
    work = _workspace(fwd_bytes, x.device)
    with _on(x.device):
        L.check(L.lib().nest_gated_ffn_forward(ct.byref(f), L.ptr(y), L.ptr(kept), L.ptr(work), fwd_bytes,
                                               L.stream_ptr(x.device)), "nest_gated_ffn_forward")
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
    with _on(x.device):
        L.check(L.lib().nest_gated_ffn_backward(ct.byref(f), L.ptr(dy), L.ptr(kept), *(L.ptr(g) for g in grads),
                                                L.ptr(work), nbytes, L.stream_ptr(x.device)), "nest_gated_ffn_backward")
    return tuple(grads)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        y, kept = gated_ffn_forward(x, w_gate, w_up, w_down, activation, training=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, w_gate, w_up, w_down, kept)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        grads = gated_ffn_backward(dy, *ctx.saved_tensors, ctx.activation, ctx.needs_input_grad[:4])
        return (*grads, None)


def gated_ffn(x, w_gate, w_up, w_down, activation: str = "silu") -> torch.Tensor:
    """gated_ffn_forward's y under autograd (x and the three weights)."""
    return _GatedFfn.apply(x, w_gate, w_up, w_down, activation)
