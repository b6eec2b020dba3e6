"""The decoder block's sizes at the limits of a launch: refused before one, on the host."""
import ctypes as ct

import pytest


@pytest.fixture(scope="module")
def L():
    from nest_splat import _lib
    return _lib


def ffn(L, rows, i, h, o, dtype):
    return L.GatedFfn(ct.sizeof(L.GatedFfn), dtype, L.ACT_SILU, i, h, o, rows, 16, 16, 16, 16)


def sizes(L, f):
    s = [ct.c_size_t() for _ in range(4)]
    return L.lib().nest_gated_ffn_sizes(ct.byref(f), *(ct.byref(v) for v in s)), [v.value for v in s]


@pytest.mark.parametrize("rows,i,h,o", [((1 << 31) - 1, 4, 4, 4), ((1 << 31) - 127, 4, 4, 4), (1 << 30, 4, 512, 4), (1 << 30, 4, 4, 1024)])
def test_more_tiles_than_a_launch_runs(L, rows, i, h, o):
    """2^31 - 1 rows are 2^23 rows of tiles, 2^32 threads; the count of them must not pass 31 bits on the way either. No
    workspace is given, so nothing here could get as far as a launch."""
    f, lib = ffn(L, rows, i, h, o, L.DTYPE_F32), L.lib()
    assert sizes(L, f)[0] == L.NEST_ERR_UNSUPPORTED and b"tiles" in lib.nest_last_error()
    assert lib.nest_gated_ffn_forward(ct.byref(f), 16, None, None, 0, None) == L.NEST_ERR_UNSUPPORTED
    for kept in (16, None):   # the backward has no product of rows by out_features
        want = L.NEST_ERR_UNSUPPORTED if o == 4 else L.NEST_ERR_WORKSPACE
        assert lib.nest_gated_ffn_backward(ct.byref(f), 16, kept, 16, 16, 16, 16, None, 0, None) == want


def test_the_largest_that_a_launch_runs(L):
    for f in (ffn(L, (1 << 31) - 512, 4, 4, 4, L.DTYPE_F32), ffn(L, (1 << 30) - 256, 4, 256, 4, L.DTYPE_F32),
              ffn(L, (1 << 31) - 1, 128, 512, 128, L.DTYPE_BF16), ffn(L, 16, 1 << 20, 1 << 20, 1 << 20, L.DTYPE_F32)):
        rc, n = sizes(L, f)
        assert rc == L.NEST_OK, (f.rows, f.hidden)
        if f.dtype == L.DTYPE_F32:
            assert n[1] >= f.rows * f.hidden * 4
