"""Values at which the decoder block's operators could go wrong, against the definitions in 64 bits: float32 products of
single terms, the ends of the types' ranges."""
import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


@pytest.fixture(scope="module")
def B():
    from nest_splat import blocks
    return blocks


def test_float32_products_of_one_term(B):
    """g = x wg of single terms, u = x and the down projection the identity, so that y is g u. Off by one unit of 2^-24 for
    the parts' products that are left out, 0.1 for the sums of the smaller five, two for the last sum (were it cut off), one
    for the product with u: 4.1. Parts that are cut off, not rounded, lose up to 7.8 units at 1 + 2^-7 - 2^-23."""
    n = 128
    g = torch.Generator().manual_seed(3)
    x, w = (1.0 + torch.rand(n, 1, generator=g) for _ in range(2))
    x[0], w[0] = 1 + 2 ** -7 - 2 ** -23, 1 + 2 ** -7 - 2 ** -23
    x[1], w[1] = 2 - 2 ** -23, 1 + 2 ** -8 - 2 ** -23
    x, w = x.to(DEV), w.to(DEV)
    y, _ = B.gated_ffn_forward(x, w, torch.ones_like(w), torch.eye(n, device=DEV), "relu")
    want = (x.double() @ w.double().T) * x.double()
    off = ((y.double() - want) / want).abs() / U
    assert float(off.max()) <= 4.25, float(off.max())


def test_float32_ends_of_the_range(B):
    """The largest numbers, past the largest bfloat16: their parts are finite and the product is what the formula gives."""
    ends = torch.tensor([3.4028234663852886e38, 3.3961775292304957e38, 3.39e38, 2.0 ** 127, 2.0 ** -100, 2.0 ** -126], device=DEV)
    x = torch.zeros(72, 8, device=DEV)
    x[:6, 0], x[6:12, 3], x[12:18, 7] = ends, -ends, ends
    wg = torch.full((40, 8), 2.0 ** -70, device=DEV)
    wg[1::2] *= -1
    wd = torch.randn(24, 40, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    y, _ = B.gated_ffn_forward(x, wg, wg * 0.75, wd, "relu")
    assert torch.isfinite(y).all()
    R.check(y, *R.ffn(x, wg, wg * 0.75, wd, "relu")["y"], "y at the ends of the range")
