"""The residual block's operators without a GPU: the library refuses what it cannot do before any launch, and reports sizes."""
import ctypes as ct

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from nest_splat import _lib
    return _lib


def layer(L, **kw):
    f = L.Linear(ct.sizeof(L.Linear), L.DTYPE_BF16, L.ACT_SILU, 0, 64, 128, 1000, 16, 16, 16, None)
    for k, v in kw.items():
        setattr(f, k, v)
    return f


def sizes(L, f):
    s = [ct.c_size_t() for _ in range(4)]
    return L.lib().nest_linear_sizes(ct.byref(f), *(ct.byref(v) for v in s)), [v.value for v in s]


def test_linear_refusals_and_sizes(L):
    lib, bad, unsup = L.lib(), L.NEST_ERR_INVALID_ARGUMENT, L.NEST_ERR_UNSUPPORTED
    for kw in (dict(struct_size=8), dict(rows=-1), dict(rows=1 << 31), dict(in_features=0), dict(out_features=(1 << 20) + 1)):
        assert sizes(L, layer(L, **kw))[0] == bad, kw
    for kw in (dict(dtype=5), dict(activation=9), dict(activation=-2), dict(rows=(1 << 31) - 1, in_features=1 << 20, out_features=1 << 20)):
        assert sizes(L, layer(L, **kw))[0] == unsup, kw
    n = 1000 * 200
    assert sizes(L, layer(L))[1][0] == 0 and sizes(L, layer(L, save8=1))[1][0] == 1000 * 128   # narrow rows make them again
    kept = lambda **kw: sizes(L, layer(L, out_features=200, **kw))[1][0]
    assert kept() == 2 * n and kept(save8=1) == n and kept(dtype=L.DTYPE_F32) == 4 * n and kept(dtype=L.DTYPE_F32, save8=1) == 2 * n
    assert kept(activation=L.ACT_RELU) == kept(activation=L.ACT_RELU, save8=1) == n and kept(activation=L.ACT_NONE) == 0
    big = layer(L, rows=4096, in_features=1024, out_features=1001)
    rc, (_, fwd, bwd, packed) = sizes(L, big)
    assert rc == L.NEST_OK and bwd >= 4096 * 1008 * 2 and packed >= bwd + 4096 * 1024 * 2
    fw = lambda f, y=16, ws=None, n=0: lib.nest_linear_forward(ct.byref(f), y, None, ws, n, None)
    split = layer(L, rows=64, in_features=8192, out_features=64)
    assert sizes(L, split)[1][1] > 0
    assert fw(split) == L.NEST_ERR_WORKSPACE and b"too small" in lib.nest_last_error()
    assert fw(big, y=None, ws=16, n=1 << 40) == bad and fw(layer(L, x=None), ws=16, n=1 << 40) == bad and fw(big, y=17, ws=16, n=1 << 40) == bad
    assert fw(layer(L, rows=0, x=None)) == L.NEST_OK
    bw = lambda f, dy=16, kept=16, codes=None, steps=None, dx=16, dw=16, db=16, ws=16, n=1 << 40: lib.nest_linear_backward(
        ct.byref(f), dy, kept, codes, steps, dx, dw, db, ws, n, None)
    assert bw(big, n=bwd - 1) == L.NEST_ERR_WORKSPACE and bw(big, codes=16, steps=16, n=packed - 1) == L.NEST_ERR_WORKSPACE
    assert bw(big, dy=None) == bad and bw(big, kept=None) == bad and bw(big, codes=16) == bad and bw(big, steps=16) == bad
    assert bw(layer(L), codes=16, steps=16, kept=None) == bad and bw(layer(L, x=None), dw=None) == bad
    from nest_splat import residual as B
    for dtype, code in ((torch.float32, L.DTYPE_F32), (torch.float16, L.DTYPE_F16), (torch.bfloat16, L.DTYPE_BF16)):
        for i, o in ((128, 128), (129, 1), (1, 129), (1, 1)):
            assert B._narrow(dtype, i, o) == (sizes(L, layer(L, dtype=code, in_features=i, out_features=o))[1][0] == 0)
    assert bw(layer(L, x=None)) == bad and bw(layer(L, weight=None)) == bad and bw(big, dx=20) == bad
    assert bw(big, dx=None, dw=None, db=None, dy=None) == L.NEST_OK


def test_pack8_refusals(L):
    lib, bad = L.lib(), L.NEST_ERR_INVALID_ARGUMENT
    for fn in (lib.nest_pack8, lib.nest_unpack8):
        call = lambda rows=4, cols=40, dt=0, x=16, c=16, s=16: fn(rows, cols, dt, x, c, s, None)
        assert call(rows=-1) == bad and call(rows=1 << 31) == bad and call(cols=0) == bad and call(cols=(1 << 20) + 1) == bad
        assert call(dt=3) == L.NEST_ERR_UNSUPPORTED and call(x=None) == bad and call(c=None) == bad and call(s=None) == bad
        assert call(rows=0, x=None, c=None, s=None) == L.NEST_OK


def test_residual_norm_refusals(L):
    lib, bad, unsup = L.lib(), L.NEST_ERR_INVALID_ARGUMENT, L.NEST_ERR_UNSUPPORTED

    def call(rows=6, cols=40, dt=0, pdt=0, x=16, h=16, gate=16, gates=1, post=16, pre=16, scale=1.0, eps=1e-6, r=16, y=16):
        return lib.nest_residual_norm(rows, cols, dt, pdt, x, h, gate, gates, post, pre, scale, eps, r, y, None, None, None)
    assert call(rows=-1) == bad and call(rows=1 << 31) == bad and call(cols=0) == bad and call(cols=8193) == bad
    assert call(dt=3) == unsup and call(dt=1, pdt=2) == unsup and call(dt=0, pdt=1) == unsup
    assert call(gates=4) == bad and call(gates=-1) == bad and call(gates=0) == bad and call(eps=-1.0) == bad and call(eps=float("nan")) == bad
    assert call(h=None) == bad and call(h=None, gate=None) == bad and call(h=None, gate=None, post=None, scale=2.0) == bad
    assert call(h=None, gate=None, post=None, pre=None) == bad
    assert call(x=None) == bad and call(r=None) == bad and call(y=None) == bad
    assert call(rows=0, x=None, r=None, y=None) == L.NEST_OK
    need = lib.nest_residual_norm_backward_workspace_size(100, 64, 0, 1)
    assert need >= 2 * 64 * 4 and lib.nest_residual_norm_backward_workspace_size(100, 64, 0, 3) == 0

    def back(rows=100, h=16, gate=16, gates=1, post=16, pre=16, scale=1.0, r=16, sp=16, sn=16, dx=16, dh=16, dg=16, dpo=16, dpr=16, ws=16, n=need):
        return lib.nest_residual_norm_backward(rows, 64, 0, 0, 16, 16, r, h, gate, gates, post, pre, scale, sp, sn, dx, dh, dg, dpo, dpr, ws, n, None)
    assert back(n=need - 1) == L.NEST_ERR_WORKSPACE and back(ws=None) == L.NEST_ERR_WORKSPACE
    for missing in ("r", "sp", "sn", "dx", "dh", "dg", "dpo", "dpr"):
        assert back(**{missing: None}) == bad, missing
    assert back(gates=3) == bad and back(gates=0) == bad and back(h=None) == bad and back(h=None, gate=None, post=None, scale=0.5) == bad


def test_embedding_refusals(L):
    lib, bad = L.lib(), L.NEST_ERR_INVALID_ARGUMENT
    call = lambda rows=4, cols=40, V=9, dt=0, ids=16, t=16, y=16: lib.nest_embedding(rows, cols, V, dt, ids, 1, t, 1.0, None, y, None)
    assert call(rows=-1) == bad and call(rows=1 << 31) == bad and call(cols=0) == bad and call(cols=(1 << 20) + 1) == bad
    assert call(V=0) == bad and call(V=(1 << 31) - 1) == bad and call(dt=3) == L.NEST_ERR_UNSUPPORTED
    assert call(ids=None) == bad and call(t=None) == bad and call(y=None) == bad and call(rows=0, ids=None, t=None, y=None) == L.NEST_OK
    need = lib.nest_embedding_backward_workspace_size(1000, 40, 9, 0)
    assert need >= 12 * 1000
    back = lambda ids=16, dy=16, dt=16, ws=16, n=need: lib.nest_embedding_backward(1000, 40, 9, 0, ids, 1, dy, 1.0, dt, ws, n, None)
    assert back(n=need - 1) == L.NEST_ERR_WORKSPACE and back(ws=None) == L.NEST_ERR_WORKSPACE
    assert back(ids=None) == bad and back(dy=None) == bad and back(dt=None) == bad


def test_tensors_on_the_host_and_arguments_that_do_not_fit_are_refused():
    from nest_splat import residual as B
    x, w = torch.zeros(2, 4), torch.zeros(4, 4)
    for call in (lambda: B.linear_forward(x, w), lambda: B.linear_backward(x, x, w), lambda: B.pack8(x), lambda: B.residual_norm_forward(x, x),
                 lambda: B.embedding_forward(torch.zeros(2, dtype=torch.int64), x), lambda: B.embedding_backward(x, torch.zeros(2, dtype=torch.int64), 3),
                 lambda: B.Packed8(torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), torch.float32),
                 lambda: B.Packed8(torch.zeros(2, 40, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), torch.float32),
                 lambda: B.residual_norm_forward(x, None), lambda: B.residual_norm_forward(x, None, scale=2.0, pre=x[0]),
                 lambda: B.residual_norm_forward(x, x, eps=-1.0), lambda: B.Linear(4, 4, activation="tanh"), lambda: B.ViewRefiner(4, 2, depth=0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: B.linear_forward(x.double(), w), lambda: B.Linear(4, 4, dtype=torch.float64), lambda: B.Embedding(4, 4, dtype="f64"),
                 lambda: B.Packed8(torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), torch.float32)):
        with pytest.raises(TypeError):
            call()
