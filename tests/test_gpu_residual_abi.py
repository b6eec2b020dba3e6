"""The residual block's operators through the C calls, with the pointers that their header allows to be left out or to be of no
bytes: a call that needs no more gives the same bits."""
import ctypes as ct

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope="module")
def L():
    from nest_splat import _lib
    return _lib


@pytest.fixture(scope="module")
def B():
    from nest_splat import residual
    return residual


def rand(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def at(t):
    return None if t is None else t.data_ptr()


def backward(L, B, dy, x, w, act=None, bias=None, kept=None, packed=None, save8=False, wants=(True, True, True), shape=None):
    """(dx, dw, db) of nest_linear_backward with the pointers given; shape: (out, in) where there is no weight."""
    O, I = shape or w.shape
    f = L.Linear(ct.sizeof(L.Linear), B._CODE[dy.dtype], B._ACT[act], int(save8), I, O, dy.shape[0], at(x), at(w), at(bias), None)
    out = [torch.full(s, float("nan"), dtype=dy.dtype, device=DEV) if n else None for s, n in zip(((dy.shape[0], I), (O, I), (O,)), wants)]
    need = ct.c_size_t()
    L.check(L.lib().nest_linear_sizes(f, None, None, None if packed else need, need if packed else None), "sizes")
    work = torch.empty(max(need.value, 1), dtype=torch.uint8, device=DEV)
    L.check(L.lib().nest_linear_backward(f, at(dy), at(kept), at(packed.codes) if packed else None, at(packed.steps) if packed else None,
                                         *(at(t) for t in out), at(work), need.value, torch.cuda.current_stream().cuda_stream), "backward")
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,out", [(24, 40), (128, 70), (24, 140)])
@pytest.mark.parametrize("from8", [False, True])
def test_linear_backward_without_the_weight(L, B, dtype, cols, out, from8):
    """The weight is read for dx and for slopes that are made again: dweight and dbias alone, without an activation, need none."""
    x, w, dy = rand(300, cols, dtype=dtype, seed=1), rand(out, cols, dtype=dtype, seed=2), rand(300, out, dtype=dtype, seed=3)
    packed = B.pack8(x) if from8 else None
    x = None if from8 else x
    _, dw, db = backward(L, B, dy, x, w, packed=packed)
    for wants in ((False, True, True), (False, True, False), (False, False, True)):
        _, dw2, db2 = backward(L, B, dy, x, None, packed=packed, wants=wants, shape=(out, cols))
        assert dw2 is None or torch.equal(dw2, dw)
        assert db2 is None or torch.equal(db2, db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,out", [(24, 40), (128, 70), (24, 140), (24, 139), (70, 200)])
@pytest.mark.parametrize("from8", [False, True])
def test_linear_backward_with_kept_of_no_bytes(L, B, dtype, cols, out, from8):
    """Where nest_linear_sizes gives kept no bytes its pointer is not looked at: here it leads to bytes that are no slopes."""
    x, w, dy = rand(300, cols, dtype=dtype, seed=1), rand(out, cols, dtype=dtype, seed=2), rand(300, out, dtype=dtype, seed=3)
    packed = B.pack8(x) if from8 else None
    x = None if from8 else x
    want = backward(L, B, dy, x, w, packed=packed)
    got = backward(L, B, dy, x, w, packed=packed, kept=torch.full((300 * out * 4,), 77, dtype=torch.uint8, device=DEV))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    if not from8 and B._narrow(dtype, cols, out):   # slopes that are made again
        want = backward(L, B, dy, x, w, "silu")
        got = backward(L, B, dy, x, w, "silu", kept=torch.full((300 * out * 4,), 77, dtype=torch.uint8, device=DEV))
        assert all(torch.equal(p, q) for p, q in zip(want, got))
