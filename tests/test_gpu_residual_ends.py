"""The residual block's operators at the ends of what their types hold and past one turn of their persistent kernels."""
import pytest
import torch

import residual_ref as R
from test_gpu_residual import B, DEV, TYPES, embed_check, linear_case, linear_check, norm_case, rand, some_ids  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- dense layer ----

@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("rows,out", [(4096, 1), (4096, 130), (16, 130)])
def test_gelu_far_below_zero_is_rounded_once(B, dtype, rows, out):
    """y of z = x alone, against half a step and what the activation's arithmetic may add: its polynomial is off by at most
    2^-16.2, two roundings of the exponent z^2 log2(e) / 2 <= 130 add 2 ln(2) 130 2^-24 = 2^-16.5, and a dozen operations 2^-20,
    together below 2^-15.  Below its type's normal numbers y may be off by half of their step, or, for bfloat16, vanish with the
    exponential."""
    x = torch.zeros(rows, 8, dtype=dtype, device=DEV)
    x[:, 0] = torch.linspace(-14.0, 4.0, rows, device=DEV).to(dtype)
    w = torch.zeros(out, 8, dtype=dtype, device=DEV)
    w[:, 0] = 1.0
    z = x[:, :1].double()
    want = (z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)).expand(rows, out)
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -15) * want.abs() + (2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126)
    for save8 in (False, True):
        y = B.linear_forward(x, w, None, "gelu", training=True, save8=save8)[0].double()
        off = (y - want).abs()
        assert (off <= bound).all(), (z.squeeze(1)[(off > bound).any(1)][:5], float((off / bound).max()))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("rows,out", [(4096, 1), (4096, 130), (16, 130)])
def test_silu_far_below_zero_is_rounded_once(B, dtype, rows, out):
    """The same of silu: the exponent z log2(e) <= 116 is rounded once and so is its factor, 2 ln(2) 116 2^-24 = 2^-16.7, and a few
    operations 2^-21, together below 2^-15."""
    x = torch.zeros(rows, 8, dtype=dtype, device=DEV)
    x[:, 0] = torch.linspace(-80.0, 4.0, rows, device=DEV).to(dtype)
    w = torch.zeros(out, 8, dtype=dtype, device=DEV)
    w[:, 0] = 1.0
    z = x[:, :1].double()
    want = (z / (1 + torch.exp(-z))).expand(rows, out)
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -15) * want.abs() + (2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126)
    off = (B.linear_forward(x, w, None, "silu")[0].double() - want).abs()
    assert (off <= bound).all(), (z.squeeze(1)[(off > bound).any(1)][:5], float((off / bound).max()))


@pytest.mark.parametrize("rows,cols,out", [(2 * 131072 + 77, 16, 32), (2 * 131072 + 129, 64, 64), (2 * 65536 + 31, 128, 128), (2 * 65536 + 65, 40, 128)])
@pytest.mark.parametrize("act", ["gelu", None])
def test_linear_narrow_past_two_turns(B, rows, cols, out, act):
    """More rows than the workgroups of a launch take in two turns (forward 1024 of 128 rows, past 128 features in and out
    together 64; backward at most 1024 of 64), the last turn partial."""
    x, w, b, r, dy = linear_case(rows, cols, out, torch.bfloat16)
    linear_check(B, x, w, b, r, dy, act)
    linear_check(B, x, w, b, r, dy, act, save8=True)


@pytest.mark.parametrize("cols,out", [(16, 64), (64, 64), (33, 50), (64, 7)])
@pytest.mark.parametrize("act,save8", [("gelu", False), ("silu", True), ("relu", False), (None, True)])
def test_linear_narrow_float32_past_two_turns(B, cols, out, act, save8):
    """The same in float32: 2048 workgroups of 64 rows forward, 512 to 1024 backward."""
    linear_check(B, *linear_case(2 * 131072 + 77, cols, out, torch.float32), act, save8)


@pytest.mark.parametrize("rows,cols,out", [(300, 40, 24), (300, 200, 140), (9, 200, 140)])
@pytest.mark.parametrize("dtype", TYPES[1:])
def test_linear_below_the_types_normal_numbers(B, dtype, rows, cols, out):
    """Gradients that are mostly below float16's 6e-5 (for bfloat16 below 1.2e-38): neither they nor their products vanish."""
    x, w, b, r, dy = linear_case(rows, cols, out, dtype)
    tiny = torch.finfo(dtype).tiny
    linear_check(B, x, w, b, r, (dy.float() * (tiny / 4)).to(dtype), None)
    if dtype is torch.float16:
        linear_check(B, x, w, b, r, (dy.float() * (tiny / 4)).to(dtype), "silu")


# ---- the residual stream between two norms ----

@pytest.mark.parametrize("dtype", TYPES)
def test_residual_norm_no_rows_and_several_gates(B, dtype):
    c = norm_case(0, 33, dtype, gates=3)
    args = [c[k] for k in ("h", "gate", "post", "pre")]
    assert args[1].shape == (3, 33)
    r, y, stats = B.residual_norm_forward(c["x"], *args)
    assert r.shape == y.shape == (0, 33)
    back = B.residual_norm_backward(c["dr"], c["dy"], r, *args, stats)
    assert back[0].shape == back[1].shape == (0, 33) and back[2].shape == (3, 33) and not any(t.any() for t in back[2:])


# ---- embedding ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [20, 3000])
def test_embedding_gradient_of_infinities_and_nan_repeats(B, rows, dtype):
    """The same bits from a second call, where what is not finite is taken out of the tiles and put back."""
    ids = some_ids(5000, rows, seed=1)
    dy = rand(5000, 48, dtype=dtype, seed=4)
    dy[::7, 3], dy[::11, 4], dy[5::13, 5], dy[::17, 3] = float("inf"), float("nan"), float("-inf"), float("-inf")
    bits = torch.int32 if dtype is torch.float32 else torch.int16
    first = B.embedding_backward(dy, ids, rows, -2.0)
    assert first.isnan().any() and first.isinf().any()
    for _ in range(3):
        assert torch.equal(first.view(bits), B.embedding_backward(dy, ids, rows, -2.0).view(bits))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(20, 48), (300, 64), (3000, 48)])
def test_embedding_gradient_below_the_types_normal_numbers(B, rows, cols, dtype):
    """Whole multiples of the type's least number, whose sums are such too: a sum of magnitudes below float32's least normal
    number is exact in any order, and so is one of float16's least numbers."""
    info = torch.finfo(dtype)
    least = float(info.smallest_normal) * float(info.eps)
    n = 700
    ids = some_ids(n, rows, seed=2)
    k = torch.randint(-3, 4, (n, cols), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    dy = (k.double() * least).to(dtype)
    assert torch.equal((dy.double() / least).long(), k)
    inside = (ids >= 0) & (ids < rows)
    want = torch.zeros(rows, cols, dtype=torch.float64, device=DEV).index_add(0, ids[inside].long(), k[inside].double()) * least
    assert torch.equal(B.embedding_backward(dy, ids, rows).double(), want.to(dtype).double())
