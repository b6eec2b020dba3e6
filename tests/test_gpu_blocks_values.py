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


def same_kind(got, want, what):
    """Infinities and NaN where the formula has them, in 16 bits."""
    got, want = got.double(), want.to(got.dtype).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), what


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [(70, 24, 20, 16), (300, 64, 100, 40), (200, 128, 300, 128), (3, 72, 77, 40), (16, 72, 75, 24),
                                  (40, 136, 132, 72), (300, 200, 1001, 136)], ids=str)
def test_infinities_with_hidden_features_that_end_inside_a_tile(B, size, dtype):
    """Positive inputs and weights, so that the formula of a row with an infinity has no NaN; what a kernel adds to the hidden
    features to fill a tile must not bring one in."""
    rows, i, h, o = size
    g = torch.Generator(device=DEV).manual_seed(5)
    x, wg, wu, wd, dy = ((torch.rand(s, generator=g, device=DEV) * 0.1 + 0.01).to(dtype) for s in ((rows, i), (h, i), (h, i), (o, h), (rows, o)))
    x[1, 3] = float("inf")
    dy[2, 5] = float("inf")
    ref = {k: v[0] for k, v in R.ffn(x, wg, wu, wd, "relu", dy).items()}
    y, kept = B.gated_ffn_forward(x, wg, wu, wd, "relu", training=True)
    same_kind(y, ref["y"], "y")
    for k in (kept, None):
        for name, v in zip(("dx", "dw_gate", "dw_up", "dw_down"), B.gated_ffn_backward(dy, x, wg, wu, wd, k, "relu")):
            same_kind(v, ref[name], (name, k is not None))
    assert torch.isinf(y[1]).all() and not torch.isnan(ref["dx"]).any()


@pytest.mark.parametrize("size", [(4, 64, 128, 64), (16, 72, 200, 40), (300, 64, 128, 64), (300, 100, 90, 128), (150, 200, 520, 136)], ids=str)
def test_float16_past_its_range_is_seen(B, size):
    """h = act(g) u is handed on in the inputs' type: past 65504 the rows it enters are infinite or NaN, though the formula's y
    would fit, never a finite number that is wrong; other rows are as they were, and bfloat16 has the range."""
    rows, i, h, o = size
    x, wg, wu, wd = (torch.rand(s, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV) for s in ((rows, i), (h, i), (h, i), (o, h)))
    x, wd = x * 0.1, wd * 2.0 ** -10
    half = [t.half() for t in (x, wg, wu, wd)]
    clean = B.gated_ffn_forward(*half, "relu")[0]
    assert torch.isfinite(clean).all()
    big = torch.ones(rows, dtype=torch.bool, device=DEV)
    big[[0, rows - 2]] = False
    x[~big] = 800.0 / i
    half[0] = x.half()
    want = R.ffn(*half, "relu")["y"][0][~big]
    y = B.gated_ffn_forward(*half, "relu")[0]
    assert (want < 65504).all() and (want / wd.half().double().sum(1) > 65504).all()
    assert torch.equal(y[big], clean[big]) and not torch.isfinite(y[~big]).any()
    bf = [t.bfloat16() for t in (x, wg, wu, wd)]
    R.check(B.gated_ffn_forward(*bf, "relu")[0], *R.ffn(*bf, "relu")["y"], "y of bfloat16")


@pytest.mark.parametrize("e", [0, 60, 100, 109, 112, 118, 126])
def test_float32_products_of_small_numbers(B, e):
    """x of 2^-e against weights of 2^e: the bound of one term, and past 2^-110, where x's last part ends below the smallest
    bfloat16, half of that, 2^-134, for x in each of g and u."""
    n = 128
    g = torch.Generator().manual_seed(4)
    x, w = ((1.0 + torch.rand(n, 1, generator=g)).to(DEV) * 2.0 ** s for s in (-e, e))
    y, _ = B.gated_ffn_forward(x, w, torch.full_like(w, 2.0 ** e), torch.eye(n, device=DEV), "relu")
    want = (x.double() @ w.double().T) * (x.double() * 2.0 ** e)
    off = ((y.double() - want) / want).abs()
    assert float(off.max()) <= 4.25 * U + 2 * 2.0 ** (e - 134)
