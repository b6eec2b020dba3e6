"""The decoder block's operators without a GPU: the library refuses what it
cannot do before any launch, reports sizes, and the generator's known answer."""
import ctypes as ct

import pytest
import torch

import block_ref as R


@pytest.fixture(scope="module")
def L():
    from nest_splat import _lib
    return _lib


def ffn(L, **kw):
    f = L.GatedFfn(ct.sizeof(L.GatedFfn), L.DTYPE_BF16, L.ACT_SILU, 64, 128, 64, 1000, 1, 1, 1, 1)
    for k, v in kw.items():
        setattr(f, k, v)
    return f


def test_norm_refusals(L):
    lib, bad, unsup = L.lib(), L.NEST_ERR_INVALID_ARGUMENT, L.NEST_ERR_UNSUPPORTED
    call = lambda rows=4, cols=8, dt=0, pdt=0, x=1, w=1, eps=1e-5, y=1: lib.nest_layer_norm(rows, cols, dt, pdt, x, w, None, eps, y, None, None, None)
    assert call(rows=-1) == bad and call(rows=1 << 31) == bad and call(cols=0) == bad and call(cols=(1 << 20) + 1) == bad
    assert call(dt=3) == unsup and call(dt=1, pdt=2) == unsup and call(dt=0, pdt=1) == unsup
    assert call(x=None) == bad and call(w=None) == bad and call(y=None) == bad and call(eps=-1.0) == bad and call(eps=float("nan")) == bad
    assert call(rows=0, x=None, y=None) == L.NEST_OK
    need = lib.nest_layer_norm_backward_workspace_size(100, 64, 0)
    assert need >= 2 * 64 * 4
    back = lambda ws, n, dw=1: lib.nest_layer_norm_backward(100, 64, 0, 0, 1, 1, 1, 1, 1, 1, dw, None, ws, n, None)
    assert back(1, need - 1) == L.NEST_ERR_WORKSPACE and b"too small" in lib.nest_last_error()
    assert back(None, need) == bad and back(1, need, dw=None) == bad


def test_dropout_refusals(L):
    lib, bad = L.lib(), L.NEST_ERR_INVALID_ARGUMENT
    call = lambda n=8, dt=0, x=1, p=0.5, y=1: lib.nest_dropout(n, dt, x, None, p, 1, 0, y, None)
    assert call(n=-1) == bad and call(p=-0.1) == bad and call(p=1.1) == bad and call(p=float("nan")) == bad
    assert call(x=None) == bad and call(y=None) == bad and call(dt=7) == L.NEST_ERR_UNSUPPORTED
    assert call(n=0, x=None, y=None) == L.NEST_OK


def test_ffn_refusals_and_sizes(L):
    lib, bad = L.lib(), L.NEST_ERR_INVALID_ARGUMENT
    sizes = lambda f: (lambda s: (lib.nest_gated_ffn_sizes(ct.byref(f), *(ct.byref(v) for v in s)), [v.value for v in s]))([ct.c_size_t() for _ in range(4)])
    for kw in (dict(struct_size=8), dict(rows=-1), dict(rows=1 << 31), dict(in_features=0), dict(hidden=0), dict(out_features=(1 << 20) + 1)):
        assert sizes(ffn(L, **kw))[0] == bad, kw
    for kw in (dict(dtype=5), dict(activation=9)):
        assert sizes(ffn(L, **kw))[0] == L.NEST_ERR_UNSUPPORTED, kw
    rc, (kept, fwd, bwd, alone) = sizes(ffn(L))
    assert rc == L.NEST_OK and alone >= bwd and alone - bwd <= kept + 256
    fw = lambda f, y=1, ws=None, n=0: lib.nest_gated_ffn_forward(ct.byref(f), y, None, ws, n, None)
    big = ffn(L, rows=4096, in_features=1024, hidden=2048, out_features=1024)
    assert sizes(big)[1][1] > 0
    assert fw(big) == L.NEST_ERR_WORKSPACE and b"too small" in lib.nest_last_error()
    assert fw(big, y=None, ws=1, n=1 << 40) == bad and fw(ffn(L, x=None), ws=1, n=1 << 40) == bad
    assert fw(ffn(L, rows=0, x=None)) == L.NEST_OK
    assert lib.nest_gated_ffn_backward(ct.byref(big), 1, None, 1, 1, 1, 1, None, 0, None) == L.NEST_ERR_WORKSPACE
    assert lib.nest_gated_ffn_backward(ct.byref(big), None, None, 1, 1, 1, 1, 1, 1 << 40, None) == bad


def test_tensors_on_the_host_are_refused():
    from nest_splat import blocks as B
    x, w = torch.zeros(2, 4), torch.zeros(4)
    with pytest.raises(ValueError):
        B.layer_norm_forward(x, w)
    with pytest.raises(ValueError):
        B.dropout_forward(x, 0.5, 1)
    with pytest.raises(ValueError):
        B.gated_ffn_forward(x, x, x, torch.zeros(4, 2))


def test_generator_known_answer():
    """The published answer of Philox 4x32-10 for a zero key and counter."""
    h = R.philox_halves([0], 0, 0)
    assert [h[2 * i] | h[2 * i + 1] << 16 for i in range(4)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    h = R.philox_halves([ones], ones, ones)
    assert [h[2 * i] | h[2 * i + 1] << 16 for i in range(4)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
