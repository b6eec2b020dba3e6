"""A residual block conditioned on the view, and its operators: a dense layer
with bias, activation and residual in its epilogue, rows held in 8 bits for its
backward pass, the residual stream between two norms, and an embedding of each
row's view (or token), each with its backward pass, on libnest_splat.

The reference has none of these; ``ViewRefiner`` runs them between the
composited feature map and the colour MLP, beside ``blocks.GatedRefiner``
(``renderer.HashINGP(refiner=...)``).

Three levels, as in ``blocks``:

- ``*_forward`` / ``*_backward``, ``pack8`` / ``unpack8``: library calls, on
  tensors;
- ``linear``, ``residual_norm``, ``embedding``: the same under autograd;
- ``Linear``, ``ResidualNorm``, ``Embedding``, ``ViewRefiner``: modules.

Tensors are on the GPU, of float32, float16 or bfloat16, with any leading
dimensions; sums are float32, run in an order that the sizes (and ids) fix, and
each result is rounded once; before that silu and gelu are off by at most 2^-15
of their value in 16 bits, and in float32 by 2^-19 of it and 2^-22 |z| (its gelu
is by erf).  linear also rounds dz = dy act'(z) to the type, as
the operand of its backward products: in 16 bits dx and dw are off by about 1.4
times what one rounding makes, and in float16 a dz past 65504 is infinite.  Its
float32 products leave out at most 2^-24 of each, and a float32 result that an
infinity enters may be NaN.  Tensors that are not contiguous are copied first.
Every call is ordered on the current stream of the tensors' device.  Gradients
of gradients are not available.
"""
from __future__ import annotations

import ctypes as ct
import math
from typing import Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .blocks import _CODE, _NAMED, _aligned, _at, _call, _code, _like, _whole, _workspace

_ACT = {None: L.ACT_NONE, "relu": L.ACT_RELU, "silu": L.ACT_SILU, "gelu": L.ACT_GELU}
_STRUCT_SIZE = ct.sizeof(L.Linear)
_GROUP = 32   # values of a row that share a step in 8 bits
MAX_NORM_COLS = 8192


# ---- rows in 8 bits ----

class Packed8:
    """Rows of x in 8 bits, as ``pack8`` makes them: ``codes`` int8 of x's shape, ``steps`` uint8 of one step for each 32
    values of a row, and the type that ``unpack8`` gives back."""

    __slots__ = ("codes", "steps", "dtype")

    def __init__(self, codes: torch.Tensor, steps: torch.Tensor, dtype: torch.dtype):
        if dtype not in _CODE:
            raise TypeError(f"dtype {dtype}: float32, float16 and bfloat16 are supported")
        if codes.dtype is not torch.int8 or steps.dtype is not torch.uint8:
            raise TypeError("codes are int8 and steps uint8")
        if codes.dim() < 1 or steps.shape != codes.shape[:-1] + (-(-codes.shape[-1] // _GROUP),):
            raise ValueError(f"steps of shape {tuple(steps.shape)} do not fit codes of {tuple(codes.shape)}")
        if codes.device != steps.device:
            raise ValueError(f"codes are on {codes.device}, steps on {steps.device}")
        if not codes.is_cuda:
            raise ValueError(f"codes are on {codes.device}: the operators run on the GPU")
        self.codes, self.steps, self.dtype = _aligned(_whole(codes)), _whole(steps), dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.steps.numel()


def pack8(x: torch.Tensor) -> Packed8:
    """x in 8 bits. 32 consecutive values of a row share a step, 2^(floor(log2 of the largest) - 6); each is held as the nearest
    whole number of steps (halves to even) within -127..127: off by at most 2^-7 of its group's largest, except that a value
    within 2^-8 of the next power of two may be off by twice that. A group with an infinity or a NaN comes back as NaN."""
    code = _code(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs a last dimension of at least 1")
    x = _whole(x)
    D = x.shape[-1]
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    steps = torch.empty(x.shape[:-1] + (-(-D // _GROUP),), dtype=torch.uint8, device=x.device)
    _call("nest_pack8", x.device, x.numel() // D, D, code, x.data_ptr(), codes.data_ptr(), steps.data_ptr())
    return Packed8(codes, steps, x.dtype)


def unpack8(packed: Packed8) -> torch.Tensor:
    """The values that ``packed`` stands for, exactly, in its type."""
    D = packed.shape[-1]
    x = torch.empty(packed.shape, dtype=packed.dtype, device=packed.device)
    _call("nest_unpack8", x.device, x.numel() // D, D, _CODE[packed.dtype], packed.codes.data_ptr(), packed.steps.data_ptr(), x.data_ptr())
    return x


# ---- dense layer ----

def _linear_struct(rows, weight, code, activation, save8):
    act = _ACT.get(activation, False)
    if act is False:
        raise ValueError(f"activation must be None or one of {sorted(k for k in _ACT if k)}, got {activation!r}")
    O, I = weight.shape
    return L.Linear(_STRUCT_SIZE, code, act, int(bool(save8)), I, O, rows)


def _slope_type(dtype, activation, save8):
    if activation == "relu":
        return torch.uint8
    if dtype is torch.float32:
        return torch.int16 if save8 else torch.float32
    return torch.uint8 if save8 else torch.int16


def _narrow(dtype, features, out_features):
    """Whether a backward makes the slopes again rather than have them kept: the library's rule."""
    return dtype is not torch.float32 and features <= 128 and out_features <= 128


def _linear_ws(f, forward=False, packed=False):
    """Bytes of a forward's workspace, or of a backward's, without or with x in 8 bits."""
    n = ct.c_size_t()
    rc = L.lib().nest_linear_sizes(f, None, n if forward else None, None if forward or packed else n, n if packed else None)
    if rc != L.NEST_OK:
        L.check(rc, "nest_linear_sizes")
    return n.value


def _matrix(weight):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("weight is an [out_features, in_features] matrix, each at least 1")
    return weight


def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                   residual: Optional[torch.Tensor] = None, training: bool = False, save8: bool = False):
    """(y, kept): y = act(x weight^T + bias) + residual for x [..., in], weight [out, in], bias [out] and residual [..., out] (or
    None), all of one type; activation None, "relu", "silu" or "gelu". ``training``: kept is what linear_backward needs of the
    activation, its slopes, of y's shape: int16 in steps of 1/26000 (float32 for float32 rows), with ``save8`` uint8 in steps of
    1/200 from -26/200 on (int16 for float32 rows), for relu always uint8. 16-bit rows of at most 128 features in and out keep
    none without ``save8``: their backward makes them again, and kept is the bias that it needs (of no elements for no bias).
    None without an activation."""
    code = _code(x, "x")
    O, I = _matrix(weight).shape
    if x.dim() < 1:
        raise ValueError("x needs a last dimension")
    if x.shape[-1] != I:
        raise ValueError(f"x has {x.shape[-1]} features, weight expects {I}")
    x = _aligned(_whole(x))
    weight = _aligned(_like(weight, x, weight.shape, "weight"))
    f = _linear_struct(x.numel() // I, weight, code, activation, save8)
    f.x, f.weight = x.data_ptr(), weight.data_ptr()
    out_shape = x.shape if O == I else x.shape[:-1] + (O,)
    if bias is not None:
        bias = _aligned(_like(bias, x, (O,), "bias"))
        f.bias = bias.data_ptr()
    if residual is not None:
        residual = _aligned(_like(residual, x, out_shape, "residual"))
        f.residual = residual.data_ptr()
    nbytes = _linear_ws(f, forward=True)
    if training:
        _linear_ws(f)   # a backward that is refused is refused here
    y = x.new_empty(out_shape)
    kept = slopes = None
    if training and activation is not None:
        if not save8 and _narrow(x.dtype, I, O):
            kept = x.new_empty(0) if bias is None else bias
        else:
            kept = slopes = torch.empty(out_shape, dtype=_slope_type(x.dtype, activation, save8), device=x.device)
    work = _workspace(nbytes, x.device)
    _call("nest_linear_forward", x.device, f, y.data_ptr(), _at(slopes), _at(work), nbytes)
    return y, kept


def linear_backward(dy: torch.Tensor, x: Union[torch.Tensor, Packed8, None], weight: torch.Tensor, kept: Optional[torch.Tensor] = None,
                    activation: Optional[str] = None, with_bias: bool = True, needs=(True, True)):
    """(dx, dweight, dbias) from dy and what the forward call kept; the residual's gradient is dy itself. x: the forward's, or
    its Packed8 (where slopes are kept), or None where neither dweight is wanted nor slopes are made again. ``needs``: whether dx
    and dweight are wanted, None else."""
    code = _code(dy, "dy")
    O, I = _matrix(weight).shape
    if dy.dim() < 1 or dy.shape[-1] != O:
        raise ValueError(f"dy of shape {tuple(dy.shape)} does not end in {O} features")
    dy = _aligned(_whole(dy))
    weight = _aligned(_like(weight, dy, weight.shape, "weight"))
    rows, in_shape = dy.numel() // O, dy.shape[:-1] + (I,)
    f = _linear_struct(rows, weight, code, activation, False)
    f.weight = weight.data_ptr()
    packed = isinstance(x, Packed8)
    if needs[1]:
        if x is None:
            raise ValueError("dweight needs x")
        if packed:
            if x.dtype is not dy.dtype or x.shape != in_shape or x.device != dy.device:
                raise ValueError(f"x in 8 bits is {x.dtype} {tuple(x.shape)} on {x.device}, expected {dy.dtype} {tuple(in_shape)} on {dy.device}")
        else:
            x = _aligned(_like(x, dy, in_shape, "x"))
            f.x = x.data_ptr()
    slopes = None
    if activation is not None:
        if kept is None:
            raise ValueError(f"the backward of {activation} needs what linear_forward(training=True) kept")
        narrow = _narrow(dy.dtype, I, O)
        full, half = (_slope_type(dy.dtype, activation, save8) for save8 in (False, True))
        if kept.device != dy.device:
            raise ValueError(f"kept is on {kept.device}, expected {dy.device}")
        if narrow and kept.dtype is dy.dtype and kept.dim() == 1 and kept.shape[0] in (0, O):
            if x is None or packed:
                raise ValueError("slopes that are not kept are made again from x: pass the tensor")
            x = _aligned(_like(x, dy, in_shape, "x"))
            kept = _aligned(_whole(kept))
            f.x = x.data_ptr()
            f.bias = kept.data_ptr() if kept.shape[0] else None
        elif kept.dtype in ((half,) if narrow else (full, half)) and kept.shape == dy.shape and kept.is_contiguous():
            f.save8 = int(kept.dtype is half)
            slopes = kept = _aligned(kept)
        else:
            raise ValueError("kept is not what linear_forward(training=True) returned for these arguments")
    use_packed = packed and needs[1]
    nbytes = _linear_ws(f, packed=use_packed)
    dx = torch.empty(in_shape, dtype=dy.dtype, device=dy.device) if needs[0] else None
    dw = torch.empty_like(weight) if needs[1] else None
    db = torch.empty(O, dtype=dy.dtype, device=dy.device) if with_bias else None
    work = _workspace(nbytes, dy.device)
    _call("nest_linear_backward", dy.device, f, dy.data_ptr(), _at(slopes),
          x.codes.data_ptr() if use_packed else None, x.steps.data_ptr() if use_packed else None, _at(dx), _at(dw), _at(db), _at(work), nbytes)
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, save8, recording):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        training = recording and (need_x or need_w or need_b)
        y, kept = linear_forward(x, weight, bias, activation, residual, training, save8)
        if training:
            codes = steps = None
            again = activation is not None and not save8 and _narrow(x.dtype, weight.shape[1], weight.shape[0])
            held = x if need_w or again else None
            if need_w and save8:
                p = pack8(x)
                held, codes, steps = None, p.codes, p.steps
            ctx.save_for_backward(held, codes, steps, weight, kept)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            x, codes, steps, weight, kept = ctx.saved_tensors
            x = Packed8(codes, steps, dy.dtype) if codes is not None else x
            dx, dw, db = linear_backward(dy, x, weight, kept, ctx.activation, need_b, (need_x, need_w))
        return dx, dw, db, dy if need_r else None, None, None, None


def linear(x, weight, bias=None, activation: Optional[str] = None, residual=None, save8: bool = False) -> torch.Tensor:
    """linear_forward's y under autograd (x, weight, bias and residual). ``save8``: the graph holds x and the slopes in 8 bits
    (float32's slopes in 16), which the weight's gradient and dz are made from."""
    return _Linear.apply(x, weight, bias, residual, activation, save8, torch.is_grad_enabled())


# ---- the residual stream between two norms ----

def _gates(x, gate):
    """How many rows of gates there are, for a gate whose shape is not a row's."""
    D = x.shape[-1]
    if gate.dim() < 1 or gate.shape[-1] != D:
        raise ValueError(f"gate of shape {tuple(gate.shape)} does not end in {D} values")
    lead = list(gate.shape[:-1])
    while lead and lead[-1] == 1:
        lead.pop()
    parts = x.dim() == 2 and len(lead) == 1 and lead[0] > 0 and x.shape[0] % lead[0] == 0
    if not parts and lead != list(x.shape[:-1][:len(lead)]):
        raise ValueError(f"gate of shape {tuple(gate.shape)} does not fit x of {tuple(x.shape)}: its leading dimensions are the first of x's")
    return gate.numel() // D


def _norm_params(x, gate, post, pre):
    """(code, parameters' code, gates, gate, post, pre): checked, contiguous, gate as [gates, cols]."""
    code = _code(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_COLS:
        raise ValueError(f"rows of 1 to {MAX_NORM_COLS} values are supported, x has shape {tuple(x.shape)}")
    row = x.shape[-1:]
    some = post if post is not None else pre if pre is not None else gate
    dtype = x.dtype if some is None else some.dtype
    if dtype is not x.dtype and dtype is not torch.float32:
        raise TypeError(f"gate, post and pre are {dtype}: float32 or the type of x ({x.dtype}) is expected")
    device = x.get_device()
    fits = lambda t: t.dtype is dtype and t.get_device() == device and t.is_contiguous()   # what _like would return as it is
    if post is not None and not (post.shape == row and fits(post)):
        post = _like(post, x, row, "post", dtype)
    if pre is not None and not (pre.shape == row and fits(pre)):
        pre = _like(pre, x, row, "pre", dtype)
    gates = 0
    if gate is not None:
        gates = 1 if gate.shape == row else _gates(x, gate)
        if not fits(gate):
            gate = _like(gate, x, gate.shape, "gate", dtype)
    return code, _CODE[dtype], gates, gate, post, pre


def residual_norm_forward(x: torch.Tensor, h: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                          post: Optional[torch.Tensor] = None, pre: Optional[torch.Tensor] = None, scale: float = 1.0, eps: float = 1e-6):
    """(r, y, stats): r = scale x + gate t with t = h / rms(h) post, and y = r / rms(r) pre, over the last dimension (at most 8192
    values); rms(v) = sqrt(mean(v^2) + eps), whose squares are summed in float32: from about 1e19 on they pass its range and the
    row's norm is zero. y is the norm of r as it is stored, in x's type.

    x is the residual stream and h a branch's output, of one shape. post [D]: the norm after the branch, None for none. pre [D]:
    the norm before the next one, None for none (y is None). gate: None, [D], or with leading dimensions that are the first of
    x's (one gate for each sequence, or for each element); for x [N, D] also [G, D], each for N / G consecutive rows. Without h,
    r is x itself. gate, post and pre are float32 or of x's type. stats: what residual_norm_backward takes, float32 [2, rows]."""
    if h is None and (gate is not None or post is not None or scale != 1.0):
        raise ValueError("without h there is no gate, no post and a scale of 1")
    if h is None and pre is None:
        raise ValueError("nothing to do without h and pre")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    code, pcode, gates, gate, post, pre = _norm_params(x, gate, post, pre)
    x = _whole(x)
    D = x.shape[-1]
    rows = x.numel() // D
    h = h if h is None else _like(h, x, x.shape, "h")
    r = x if h is None else torch.empty_like(x)
    y = None if pre is None else torch.empty_like(x)
    stats = x.new_empty((2, rows), dtype=torch.float32)
    if rows == 0:   # whose tensors have no addresses to tell them from those left out
        return r, y, stats
    at = stats.data_ptr()
    _call("nest_residual_norm", x.device, rows, D, code, pcode, x.data_ptr(), _at(h), _at(gate), gates, _at(post), _at(pre), scale, eps,
          r.data_ptr(), _at(y), at, at + 4 * rows)
    return r, y, stats


def residual_norm_backward(dr: Optional[torch.Tensor], dy: Optional[torch.Tensor], r: torch.Tensor, h: Optional[torch.Tensor] = None,
                           gate: Optional[torch.Tensor] = None, post: Optional[torch.Tensor] = None, pre: Optional[torch.Tensor] = None,
                           stats: Optional[torch.Tensor] = None, scale: float = 1.0):
    """(dx, dh, dgate, dpost, dpre) from the gradients of r and y (None: zero) and what residual_norm_forward returned; a
    gradient whose input is None is None. dgate has gate's shape."""
    if h is None and (gate is not None or post is not None or scale != 1.0):
        raise ValueError("without h there is no gate, no post and a scale of 1")
    if dy is not None and pre is None:
        raise ValueError("without pre there is no y, and no dy")
    code, pcode, gates, gate, post, pre = _norm_params(r, gate, post, pre)
    r = _whole(r)
    D = r.shape[-1]
    rows = r.numel() // D
    dr = dr if dr is None else _like(dr, r, r.shape, "dr")
    dy = dy if dy is None else _like(dy, r, r.shape, "dy")
    h = h if h is None else _like(h, r, r.shape, "h")
    if stats is None:
        raise ValueError("stats is missing: residual_norm_forward returns it")
    stats = _like(stats, r, (2, rows), "stats", torch.float32)
    dx = torch.empty_like(r)
    dh = None if h is None else torch.empty_like(r)
    dgate, dpost, dpre = (None if t is None else torch.empty_like(t) if rows else torch.zeros_like(t) for t in (gate, post, pre))
    if rows == 0:
        return dx, dh, dgate, dpost, dpre
    nbytes = L.lib().nest_residual_norm_backward_workspace_size(rows, D, code, gates)
    work = _workspace(nbytes, r.device)
    at = stats.data_ptr()
    _call("nest_residual_norm_backward", r.device, rows, D, code, pcode, _at(dr), _at(dy), r.data_ptr(), _at(h), _at(gate), gates, _at(post),
          _at(pre), scale, at, at + 4 * rows, dx.data_ptr(), _at(dh), _at(dgate), _at(dpost), _at(dpre), _at(work), nbytes)
    return dx, dh, dgate, dpost, dpre


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post, pre, scale, eps):
        r, y, stats = residual_norm_forward(x, h, gate, post, pre, scale, eps)
        ctx.save_for_backward(r, h, gate, post, pre, stats)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if h is None:
            return y
        return r if y is None else (r, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, first, second=None):
        r, h, gate, post, pre, stats = ctx.saved_tensors
        dr, dy = (None, first) if h is None else (first, second)
        if dr is None and dy is None:
            return (None,) * 7
        return (*residual_norm_backward(dr, dy, r, h, gate, post, pre, stats, ctx.scale), None, None)


def residual_norm(x, h=None, gate=None, post=None, pre=None, scale: float = 1.0, eps: float = 1e-6):
    """residual_norm_forward's (r, y) under autograd (x, h, gate, post and pre); y is None without pre, r is x without h."""
    out = _ResidualNorm.apply(x, h, gate, post, pre, scale, eps)
    if h is None:
        return x, out
    return (out, None) if pre is None else out


# ---- embedding ----

def _id_args(ids):
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids are {ids.dtype}: int32 and int64 are supported")
    return _whole(ids), int(ids.dtype is torch.int64)


def embedding_forward(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = residual + scale table[ids] for ids (int32 or int64) of any shape, table [rows, D] and residual [*ids.shape, D] or None.
    An id outside the table (-1, say, for no view) adds nothing."""
    code = _code(table, "table")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("table is a [rows, D] matrix, each at least 1")
    ids, wide = _id_args(ids)
    if ids.get_device() != table.get_device():
        raise ValueError(f"ids are on {ids.device}, expected {table.device}")
    V, D = table.shape
    table = _whole(table)
    shape = ids.shape + (D,)
    if residual is not None:
        residual = _like(residual, table, shape, "residual")
    y = torch.empty(shape, dtype=table.dtype, device=table.device)
    _call("nest_embedding", table.device, ids.numel(), D, V, code, ids.data_ptr(), wide, table.data_ptr(), scale, _at(residual), y.data_ptr())
    return y


def embedding_backward(dy: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    """dtable [rows, D]: scale times the sum of dy [*ids.shape, D] over the places of each id, in dy's type; the sums run in an
    order that the sizes and ids fix, so results repeat bit for bit. The residual's gradient is dy itself."""
    code = _code(dy, "dy")
    ids, wide = _id_args(ids)
    if ids.get_device() != dy.get_device():
        raise ValueError(f"ids are on {ids.device}, expected {dy.device}")
    if dy.dim() < 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] < 1:
        raise ValueError(f"dy of shape {tuple(dy.shape)} does not fit ids of {tuple(ids.shape)}")
    dy = _whole(dy)
    N, D, rows = ids.numel(), dy.shape[-1], int(rows)
    if rows < 1:
        raise ValueError(f"the table needs at least one row, got {rows}")
    dtable = torch.empty((rows, D), dtype=dy.dtype, device=dy.device)
    nbytes = L.lib().nest_embedding_backward_workspace_size(N, D, rows, code) if N else 0
    work = _workspace(nbytes, dy.device)
    _call("nest_embedding_backward", dy.device, N, D, rows, code, ids.data_ptr(), wide, dy.data_ptr(), scale, dtable.data_ptr(), _at(work), nbytes)
    return dtable


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, residual):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return embedding_forward(ids, table, scale, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dtable = embedding_backward(dy, *ctx.saved_tensors, ctx.rows, ctx.scale) if ctx.needs_input_grad[1] else None
        return None, dtable, None, dy if ctx.needs_input_grad[3] else None


def embedding(ids, table, scale: float = 1.0, residual=None) -> torch.Tensor:
    """embedding_forward under autograd (table and residual)."""
    return _Embedding.apply(ids, table, scale, residual)


# ---- modules ----

def _type(dtype):
    t = _NAMED.get(dtype, dtype)
    if t not in _CODE:
        raise TypeError(f"dtype {dtype!r}: float32, float16 and bfloat16 are supported")
    return t


class Linear(nn.Module):
    """linear with float32 weight and bias, computed in ``dtype`` (x, the parameters and the residual are cast to it, y has it)."""

    def __init__(self, features: int, out_features: int, bias: bool = True, activation: Optional[str] = None, dtype="bf16",
                 save8: bool = False, seed: int = 0):
        super().__init__()
        if activation not in _ACT:
            raise ValueError(f"activation must be None or one of {sorted(k for k in _ACT if k)}, got {activation!r}")
        self.activation, self.dtype, self.save8 = activation, _type(dtype), bool(save8)
        g = torch.Generator().manual_seed(seed)
        bound = math.sqrt(3.0 / features)
        self.weight = nn.Parameter((torch.rand((out_features, features), generator=g) * 2 - 1) * bound)
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        t = self.dtype
        return linear(x.to(t), self.weight.to(t), None if self.bias is None else self.bias.to(t), self.activation,
                      None if residual is None else residual.to(t), self.save8)


class ResidualNorm(nn.Module):
    """residual_norm with float32 parameters: (r, y) of the stream x and a branch h of any of the types.

    ``gate``: the value that a learned gate of each channel starts at, None for none. ``post`` and ``pre``: whether the branch and
    the new stream are normed; y is None without ``pre``."""

    def __init__(self, features: int, gate: Optional[float] = 1.0, post: bool = True, pre: bool = True, scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        self.scale, self.eps = float(scale), float(eps)
        self.gate = None if gate is None else nn.Parameter(torch.full((features,), float(gate)))
        self.post = nn.Parameter(torch.ones(features)) if post else None
        self.pre = nn.Parameter(torch.ones(features)) if pre else None

    def forward(self, x: torch.Tensor, h: torch.Tensor):
        return residual_norm(x, h, self.gate, self.post, self.pre, self.scale, self.eps)


class Embedding(nn.Module):
    """embedding with a float32 table that starts at zero, computed in ``dtype``."""

    def __init__(self, rows: int, features: int, scale: float = 1.0, dtype="bf16"):
        super().__init__()
        self.scale, self.dtype = float(scale), _type(dtype)
        self.weight = nn.Parameter(torch.zeros(rows, features))

    def forward(self, ids: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        t = self.dtype
        return embedding(ids, self.weight.to(t), self.scale, None if residual is None else residual.to(t))


class ViewRefiner(nn.Module):
    """``depth`` residual blocks over the feature channels of every pixel, conditioned on the view that the pixel belongs to.

    An embedding of the view is added to the stream; each block is two dense layers between a norm before and a norm after,
    joined to the stream by a gate of each channel. The rows run through the blocks in ``dtype``; with ``save8`` the dense layers
    keep 8 bits of what their backward passes need. The table and the gates start at zero, so a new refiner returns its input
    rounded to dtype. ``seed`` makes the weights."""

    def __init__(self, features: int, views: int, hidden: Optional[int] = None, depth: int = 1, activation: str = "gelu", dtype="bf16",
                 save8: bool = False, seed: int = 0):
        super().__init__()
        if depth < 1:
            raise ValueError(f"depth must be at least 1, got {depth}")
        self.features, self.views, self.dtype = int(features), int(views), _type(dtype)
        hidden = hidden or 2 * features
        self.embed = Embedding(views, features, dtype=dtype)
        self.first = nn.Parameter(torch.ones(features))   # the norm before the first block
        self.ups = nn.ModuleList(Linear(features, hidden, True, activation, dtype, save8, seed + 2 * k) for k in range(depth))
        self.downs = nn.ModuleList(Linear(hidden, features, True, None, dtype, save8, seed + 2 * k + 1) for k in range(depth))
        self.joins = nn.ModuleList(ResidualNorm(features, gate=0.0, pre=k + 1 < depth) for k in range(depth))

    def forward(self, x: torch.Tensor, views: Union[None, int, torch.Tensor] = None) -> torch.Tensor:
        """x [..., features] of any of the types -> the same shape and type. views: the view of each row (an integer tensor of
        x's leading dimensions, -1 for none), of all rows, or None."""
        if x.shape[-1] != self.features:
            raise ValueError(f"expected {self.features} feature channels, got {x.shape[-1]}")
        r = x.to(self.dtype)
        if views is not None:
            if not isinstance(views, torch.Tensor):
                if not 0 <= int(views) < self.views:
                    raise ValueError(f"view {views} of {self.views}")
                views = torch.full(x.shape[:-1], int(views), dtype=torch.int32, device=x.device)
            if views.shape != x.shape[:-1]:
                raise ValueError(f"views of shape {tuple(views.shape)} for rows of {tuple(x.shape[:-1])}")
            r = self.embed(views, r)
        y = residual_norm(r, pre=self.first)[1]
        for up, down, join in zip(self.ups, self.downs, self.joins):
            r, y = join(r, down(up(y)))
        return r.to(x.dtype)

    def refine_image(self, color: torch.Tensor, view: Union[None, int] = None) -> torch.Tensor:
        """A feature map [C, H, W] refined pixel by pixel, as a pixel of ``view`` (None: of none)."""
        C, H, W = color.shape
        return self(color.reshape(C, -1).t(), view).t().reshape(C, H, W).contiguous()
