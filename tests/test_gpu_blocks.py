"""The decoder block's operators (nest_splat.blocks) against the formulas in
64 bits: values and gradients within the element-wise bounds of block_ref.py,
at the sizes, layouts and values where they can go wrong."""
import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope="module")
def B():
    from nest_splat import blocks
    return blocks


def rand(*shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)


# ---- layer norm ----

def norm_case(rows, cols, dtype, pdt, seed=1, shift=0.3):
    return (rand(rows, cols, dtype=dtype, seed=seed, shift=shift), rand(cols, dtype=pdt, seed=seed + 1, scale=0.2, shift=1.0),
            rand(cols, dtype=pdt, seed=seed + 2, scale=0.3), rand(rows, cols, dtype=dtype, seed=seed + 3))


def norm_check(B, x, w, b, dy, eps=1e-5):
    ref = R.norm(x.reshape(-1, x.shape[-1]), w, b, eps, dy.reshape(-1, x.shape[-1]))
    y, mean, rstd = B.layer_norm_forward(x, w, b, eps)
    dx, dw, db = B.layer_norm_backward(dy, x, w, mean, rstd, with_bias=b is not None)
    got = {"y": y, "dx": dx, "dw": dw, "db": db}
    for k, v in got.items():
        if v is None:
            assert k == "db" and b is None
            continue
        assert v.dtype == (x.dtype if k in ("y", "dx") else w.dtype)
        R.check(v.reshape(ref[k][0].shape), *ref[k], f"{k} of {tuple(x.shape)} {x.dtype} {w.dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 2048), (70, 7), (513, 64), (37, 129), (1030, 16), (9, 515), (5, 1024),
                                       (6, 1031), (3, 2049), (2, 4100), (3, 8200), (2, 16400), (1100, 520)])
def test_norm_values_and_gradients(B, rows, cols, dtype):
    norm_check(B, *norm_case(rows, cols, dtype, dtype))


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_norm_float32_parameters(B, dtype):
    norm_check(B, *norm_case(41, 200, dtype, torch.float32))
    x, w, _, dy = norm_case(41, 200, dtype, torch.float32)
    norm_check(B, x, w, None, dy)


def test_norm_constant_rows_large_means_and_other_eps(B):
    x, w, b, dy = norm_case(8, 96, torch.float32, torch.float32)
    x[0] = 3.0
    x[1] = 0.0
    x[2] += 1000.0
    norm_check(B, x, w, b, dy)
    norm_check(B, x[3:], w, b, dy[3:], eps=0.1)


def test_norm_nan_and_infinity_stay_in_their_rows(B):
    x, w, b, _ = norm_case(9, 130, torch.float32, torch.float32)
    clean = B.layer_norm_forward(x, w, b)[0]
    x[2, 5], x[7, 129] = float("nan"), float("inf")
    y = B.layer_norm_forward(x, w, b)[0]
    rows = torch.ones(9, dtype=torch.bool)
    rows[[2, 7]] = False
    assert torch.equal(y[rows.to(DEV)], clean[rows.to(DEV)])
    assert torch.isnan(y[2]).all() and torch.isnan(y[7]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_no_rows(B, dtype):
    x, w, b, dy = norm_case(0, 33, dtype, dtype)
    y, mean, rstd = B.layer_norm_forward(x, w, b)
    assert y.shape == (0, 33) and mean.numel() == 0
    dx, dw, db = B.layer_norm_backward(dy, x, w, mean, rstd)
    assert dx.shape == (0, 33) and not dw.any() and not db.any()


def test_norm_strides_leading_dimensions_and_alignment(B):
    w, b = rand(24, dtype=torch.float16, seed=5), rand(24, dtype=torch.float16, seed=6)
    wide = rand(24, 6, 10, dtype=torch.float16, seed=7)
    x = wide.permute(1, 2, 0)  # channels first in memory
    dy = rand(6, 10, 24, dtype=torch.float16, seed=8)
    norm_check(B, x, w, b, dy)
    flat = rand(1 + 7 * 24, dtype=torch.float16, seed=9)
    norm_check(B, flat[1:].view(7, 24), w, b, rand(7, 24, dtype=torch.float16, seed=10))  # 2-byte aligned
    norm_check(B, rand(9, 30, dtype=torch.float16, seed=11)[:, 3:27], w, b, rand(9, 24, dtype=torch.float16, seed=12))


def test_norm_repeats_bit_for_bit_and_autograd(B):
    x, w, b, dy = norm_case(5000, 96, torch.bfloat16, torch.bfloat16)
    y, mean, rstd = B.layer_norm_forward(x, w, b)
    first = B.layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(first, B.layer_norm_backward(dy, x, w, mean, rstd)))
    ps = [t.clone().requires_grad_() for t in (x, w, b)]
    out = B.layer_norm(*ps)
    assert torch.equal(out, y)
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(out, ps, dy)))


# ---- dropout ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 4099])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_is_the_generator_exactly(B, n, dtype, residual):
    x, r = rand(n, dtype=dtype, seed=n), rand(n, dtype=dtype, seed=n + 1)
    seed, offset, p = 0xFEDCBA9876543210, (5 << 32) + n, 0.37
    drop, scale = R.dropped(n, p, seed, offset)
    want = torch.where(drop, torch.zeros(()), x.cpu().float() * torch.tensor(scale, dtype=torch.float32))
    if residual:
        want = r.cpu().float() + want
    got = B.dropout_forward(x, p, seed, offset, residual=r if residual else None)
    assert torch.equal(got.cpu(), want.to(dtype))
    back = B.dropout_backward(x, p, seed, offset)
    assert torch.equal(back.cpu(), torch.where(drop, torch.zeros(()), x.cpu().float() * torch.tensor(scale, dtype=torch.float32)).to(dtype))


def test_dropout_ends_of_p_and_values_that_are_not_finite(B):
    x = rand(1000, dtype=torch.float32, seed=3)
    assert torch.equal(B.dropout_forward(x, 0.0, 1), x)
    bad = torch.full((1000,), float("nan"), device=DEV)
    bad[::2] = float("inf")
    assert not B.dropout_forward(bad, 1.0, 1).any()
    assert torch.equal(B.dropout_forward(bad, 1.0, 1, residual=x), x)
    drop, _ = R.dropped(1000, 0.5, 9, 0)
    y = B.dropout_forward(bad, 0.5, 9)
    assert not y[drop.to(DEV)].any() and not torch.isfinite(y[~drop.to(DEV)]).any()


def test_dropout_share_offsets_and_seeds(B):
    x = torch.ones(1 << 20, device=DEV)
    a, b, c = B.dropout_forward(x, 0.3, 7, 0), B.dropout_forward(x, 0.3, 7, 1), B.dropout_forward(x, 0.3, 8, 0)
    for t in (a, b, c):  # the share's standard deviation is 4.5e-4: six of them
        assert abs(float((t == 0).double().mean()) - 0.3) < 2.7e-3
    for s, t in ((a, b), (a, c), (b, c)):  # both dropped: 0.09 with a deviation of 2.8e-4
        assert abs(float(((s == 0) & (t == 0)).double().mean()) - 0.09) < 1.7e-3


def test_dropout_past_2_31_elements(B):
    n = (1 << 31) + 77
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = B.dropout_forward(x, 0.25, 11, 2)
    at = ((1 << 31) - 40) // 8
    drop, _ = R.dropped(n - at * 8, 0.25, 11, 2, first_block=at)
    assert torch.equal((y[at * 8:] == 0).cpu(), drop)


def test_dropout_strides_alignment_and_autograd(B):
    base = rand(40, 30, dtype=torch.float16, seed=4)
    x = base.t()
    assert torch.equal(B.dropout_forward(x, 0.2, 5), B.dropout_forward(x.contiguous(), 0.2, 5))
    flat = rand(1001, dtype=torch.float16, seed=4)
    assert torch.equal(B.dropout_forward(flat[1:], 0.2, 5), B.dropout_forward(flat[1:].clone(), 0.2, 5))
    a, r = rand(50, 33, dtype=torch.float32, seed=1).requires_grad_(), rand(50, 33, dtype=torch.float32, seed=2).requires_grad_()
    y = B.dropout(a, 0.4, 21, 3, r)
    dy = rand(50, 33, dtype=torch.float32, seed=3)
    da, dr = torch.autograd.grad(y, (a, r), dy)
    assert torch.equal(da, B.dropout_backward(dy, 0.4, 21, 3)) and torch.equal(dr, dy)


# ---- gated feed-forward ----

def ffn_case(rows, i, h, o, dtype, seed=1):
    s = (2.0 / (i + h)) ** 0.5
    return (rand(rows, i, dtype=dtype, seed=seed), rand(h, i, dtype=dtype, seed=seed + 1, scale=s), rand(h, i, dtype=dtype, seed=seed + 2, scale=s),
            rand(o, h, dtype=dtype, seed=seed + 3, scale=s), rand(rows, o, dtype=dtype, seed=seed + 4))


def ffn_check(B, x, wg, wu, wd, dy, kind):
    what = f"{x.shape[0]}x{x.shape[1]}, {wg.shape[0]}, {wd.shape[0]} {x.dtype} {kind}"
    ref = R.ffn(x, wg, wu, wd, kind, dy)
    y, kept = B.gated_ffn_forward(x, wg, wu, wd, kind, training=True)
    R.check(y, *ref["y"], "y of " + what)
    alone, none = B.gated_ffn_forward(x, wg, wu, wd, kind)
    assert none is None
    R.check(alone, *ref["y"], "y alone of " + what)
    for k in (kept, None):
        grads = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), B.gated_ffn_backward(dy, x, wg, wu, wd, k, kind)))
        for name, v in grads.items():
            R.check(v, *ref[name], f"{name} of {what}, kept {k is not None}")


FFN_SIZES = [(1, 1, 1, 1), (1, 8, 16, 8), (2, 5, 3, 7), (17, 64, 128, 64), (100, 16, 64, 16), (1000, 32, 128, 32), (513, 48, 200, 48),
             (300, 128, 512, 128), (1, 512, 1024, 512), (3, 515, 1365, 515), (16, 256, 768, 256), (33, 264, 520, 136), (260, 131, 263, 129),
             (200, 520, 1000, 264), (129, 64, 640, 64), (700, 17, 33, 19), (640, 256, 512, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", FFN_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_ffn_values_and_gradients(B, size, dtype):
    kind = ("silu", "gelu", "relu")[(FFN_SIZES.index(size) + TYPES.index(dtype)) % 3]
    ffn_check(B, *ffn_case(*size, dtype), kind)


# Rows of at most 128 features: every padded width, every number of waves that share the hidden features, hidden
# features past one launch of the backward and past the forward's LDS, unlike widths, the last rows of a workgroup.
NARROW_SIZES = [(64, 16, 20, 16), (65, 33, 30, 40), (100, 64, 60, 33), (777, 96, 32, 96), (129, 128, 64, 100), (2100, 32, 256, 8),
                (300, 64, 256, 64), (90, 40, 300, 64), (333, 128, 256, 128), (200, 96, 400, 72), (150, 5, 700, 128), (4099, 24, 96, 24)]


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("size", NARROW_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_ffn_narrow_rows(B, size, dtype):
    kind = ("silu", "gelu", "relu")[(NARROW_SIZES.index(size) + TYPES.index(dtype)) % 3]
    ffn_check(B, *ffn_case(*size, dtype), kind)


FEW_ROWS = [1, 2, 4, 5, 8, 9, 16, 17, 31, 32, 33]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", FEW_ROWS)
def test_ffn_few_rows(B, rows, dtype):
    """Each way of dealing k to lanes and waves, with odd and even lengths of it."""
    i, h, o = (264, 520, 200) if rows % 2 else (301, 2060, 77)
    ffn_check(B, *ffn_case(rows, i, h, o, dtype), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", range(1, 10))
def test_ffn_every_count_of_steps(B, steps, dtype):
    """Sums of 1 to 9 steps of 128 bytes, the last one short: each way in and out of two and four LDS buffers."""
    n = steps * (32 if dtype is torch.float32 else 64)
    ffn_check(B, *ffn_case(n - 1, n - 5, n - 3, 136, dtype), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1500, 200, 1400, 136), (3000, 140, 2000, 132)], ids=lambda s: "x".join(map(str, s)))
def test_ffn_many_tiles(B, size, dtype):
    """More tiles than run at once, at sizes whose sides end inside a tile."""
    ffn_check(B, *ffn_case(*size, dtype), "gelu")


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_ffn_activations_over_their_range(B, dtype, kind):
    """One input feature from -30 to 30 through gate weights of 1: the pre-activations are the inputs."""
    x = torch.linspace(-30, 30, 257, device=DEV).to(dtype)[:, None].repeat(1, 8) / 8
    one = torch.ones(16, 8, device=DEV, dtype=dtype)
    ffn_check(B, x, one, one * 0.5, torch.ones(8, 16, device=DEV, dtype=dtype), rand(257, 8, dtype=dtype, seed=2), kind)


@pytest.mark.parametrize("dtype", TYPES)
def test_ffn_no_rows(B, dtype):
    x, wg, wu, wd, dy = ffn_case(0, 24, 40, 16, dtype)
    y, kept = B.gated_ffn_forward(x, wg, wu, wd, training=True)
    assert y.shape == (0, 16)
    dx, *dws = B.gated_ffn_backward(dy, x, wg, wu, wd, kept)
    assert dx.shape == (0, 24) and all(w.shape == d.shape and not d.any() for w, d in zip((wg, wu, wd), dws))


@pytest.mark.parametrize("rows", [4, 150, 3000])
def test_ffn_nan_and_infinity_stay_in_their_rows(B, rows):
    x, wg, wu, wd, dy = ffn_case(rows, 64, 128, 64, torch.bfloat16)
    clean = B.gated_ffn_forward(x, wg, wu, wd)[0]
    cx = B.gated_ffn_backward(dy, x, wg, wu, wd)[0]
    x[1, 3], x[3, 63] = float("nan"), float("inf")
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[[1, 3]] = False
    y = B.gated_ffn_forward(x, wg, wu, wd)[0]
    dx = B.gated_ffn_backward(dy, x, wg, wu, wd)[0]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cx[keep])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any()


@pytest.mark.parametrize("size", [(40, 72, 136, 72), (900, 32, 64, 32)], ids=str)
def test_ffn_strides_leading_dimensions_and_alignment(B, size):
    rows, i, h, o = size
    x, wg, wu, wd, dy = ffn_case(rows, i, h, o, torch.float16)
    want = B.gated_ffn_forward(x, wg, wu, wd)[0]
    assert torch.equal(B.gated_ffn_forward(x.t().contiguous().t(), wg, wu.t().contiguous().t(), wd)[0], want)
    assert torch.equal(B.gated_ffn_forward(x.view(4, rows // 4, i), wg, wu, wd)[0].view(rows, o), want)

    def shifted(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    ffn_check(B, *(shifted(t) for t in (x, wg, wu, wd, dy)), "silu")


@pytest.mark.parametrize("size", [(5, 64, 128, 64), (2000, 64, 128, 64), (300, 256, 512, 256)], ids=str)
def test_ffn_repeats_autograd_and_wanted_gradients(B, size):
    x, wg, wu, wd, dy = ffn_case(*size, torch.bfloat16)
    y, kept = B.gated_ffn_forward(x, wg, wu, wd, "gelu", training=True)
    first = B.gated_ffn_backward(dy, x, wg, wu, wd, kept, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(first, B.gated_ffn_backward(dy, x, wg, wu, wd, kept, "gelu")))
    ps = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    out = B.gated_ffn(*ps, "gelu")
    assert torch.equal(out, y)
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(out, ps, dy)))
    for k in range(4):
        needs = [j == k for j in range(4)]
        got = B.gated_ffn_backward(dy, x, wg, wu, wd, kept, "gelu", needs)
        assert [t is not None for t in got] == needs and torch.equal(got[k], first[k])


# ---- differences, streams, graphs ----

def test_gradients_against_differences(B):
    """Along a random direction, the loss c . f: a central difference of step e = 2^-7 of f in float32 is off by e^2 of the
    third derivative and by about 2^-24 |c| |f| / e; both are under 2e-3 of these gradients' size."""
    x, w, b, c = norm_case(20, 48, torch.float32, torch.float32)
    ffn = ffn_case(20, 48, 96, 48, torch.float32)[1:4]
    e = 2.0 ** -7
    for f, args in ((lambda x, w, b: B.layer_norm(x, w, b), (x, w, b)), (lambda x, *ws: B.gated_ffn(x, *ws, "silu"), (x, *ffn)),
                    (lambda x, *ws: B.gated_ffn(x, *ws, "gelu"), (x, *ffn)), (lambda x, r: B.dropout(x, 0.3, 4, 0, r), (x, c))):
        args = [a.clone().requires_grad_() for a in args]
        grads = torch.autograd.grad((f(*args) * c).sum(), args)
        for k, (a, g) in enumerate(zip(args, grads)):
            v = rand(*a.shape, dtype=torch.float32, seed=50 + k)
            v = v * (a.detach().norm() / v.norm() * 0.1)
            with torch.no_grad():
                lo, hi = ((f(*(t + s * e * v if j == k else t for j, t in enumerate(args))).double() * c.double()).sum() for s in (-1, 1))
            diff, exact = float((hi - lo) / (2 * e)), float((g.double() * v.double()).sum())
            assert abs(diff - exact) <= 2e-3 * float(g.double().norm() * v.double().norm()), (k, diff, exact)


def test_another_stream_and_graph_replays(B):
    x, w, b, dy = norm_case(700, 64, torch.bfloat16, torch.bfloat16)
    ws = ffn_case(700, 64, 128, 64, torch.bfloat16)[1:4]

    def step():
        n, mean, rstd = B.layer_norm_forward(x, w, b)
        f, kept = B.gated_ffn_forward(n, *ws, "silu", training=True)
        y = B.dropout_forward(f, 0.1, 3, 4, residual=x)
        df = B.dropout_backward(dy, 0.1, 3, 4)
        dn, *dws = B.gated_ffn_backward(df, n, *ws, kept, "silu")
        return [y, *dws, *B.layer_norm_backward(dn, x, w, mean, rstd)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(rand(700, 64, dtype=torch.bfloat16, seed=90 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), k


# ---- refusals ----

def test_refusals(B):
    x, w, b, dy = norm_case(4, 32, torch.float16, torch.float16)
    ws = ffn_case(4, 32, 48, 32, torch.float16)[1:4]
    y, mean, rstd = B.layer_norm_forward(x, w, b)
    _, kept = B.gated_ffn_forward(x, *ws, training=True)
    for error, call in [
            (TypeError, lambda: B.layer_norm_forward(x.double(), w, b)),
            (TypeError, lambda: B.layer_norm_forward(x, w.bfloat16(), b)),
            (TypeError, lambda: B.layer_norm_forward(x, w, b.float())),
            (ValueError, lambda: B.layer_norm_forward(x, w[:31], b)),
            (ValueError, lambda: B.layer_norm_forward(x, w, b.cpu())),
            (ValueError, lambda: B.layer_norm_forward(x.cpu(), w, b)),
            (ValueError, lambda: B.layer_norm_forward(x, w, b, eps=-1.0)),
            (ValueError, lambda: B.layer_norm_forward(x[:, :0], w[:0], None)),
            (ValueError, lambda: B.layer_norm_backward(dy[:3], x, w, mean, rstd)),
            (TypeError, lambda: B.layer_norm_backward(dy, x, w, mean.half(), rstd)),
            (ValueError, lambda: B.dropout_forward(x, 1.5, 1)),
            (ValueError, lambda: B.dropout_forward(x, float("nan"), 1)),
            (ValueError, lambda: B.dropout_forward(x, 0.5, -1)),
            (ValueError, lambda: B.dropout_forward(x, 0.5, 1, 1 << 64)),
            (ValueError, lambda: B.dropout_forward(x, 0.5, 1, residual=x[:2])),
            (TypeError, lambda: B.dropout_forward(x.long(), 0.5, 1)),
            (ValueError, lambda: B.gated_ffn_forward(x, *ws, activation="tanh")),
            (ValueError, lambda: B.gated_ffn_forward(x[:, :31], *ws)),
            (ValueError, lambda: B.gated_ffn_forward(x, ws[0], ws[1][:40], ws[2])),
            (TypeError, lambda: B.gated_ffn_forward(x, ws[0].float(), ws[1], ws[2])),
            (ValueError, lambda: B.gated_ffn_backward(dy[:, :16], x, *ws, kept)),
            (ValueError, lambda: B.gated_ffn_backward(dy, x, *ws, torch.zeros(5, dtype=torch.uint8, device=DEV)))]:
        with pytest.raises(error):
            call()
    a = x.clone().requires_grad_()
    g, = torch.autograd.grad(B.layer_norm(a, w, b).float().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- modules and the path that runs them together ----

def test_modules_against_the_definitions(B):
    torch.manual_seed(0)
    norm = B.LayerNorm(48).to(DEV)
    with torch.no_grad():
        norm.weight.normal_(1, 0.2)
        norm.bias.normal_(0, 0.2)
    x = rand(5, 7, 48, dtype=torch.float16, seed=1)
    ref = R.norm(x.view(-1, 48), norm.weight.detach(), norm.bias.detach(), 1e-5)
    R.check(norm(x).detach().view(-1, 48), *ref["y"], "LayerNorm")
    ffn = B.GatedFFN(48, 96, 40, "gelu", "f16").to(DEV)
    ws = [w.detach().half() for w in (ffn.w_gate, ffn.w_up, ffn.w_down)]
    y = ffn(x.float())
    assert y.shape == (5, 7, 40) and y.dtype == torch.float16
    R.check(y.detach().view(-1, 40), *R.ffn(x.view(-1, 48), *ws, "gelu")["y"], "GatedFFN")
    y.sum().backward()
    assert all(w.grad is not None and w.grad.dtype == torch.float32 and w.grad.any() for w in ffn.parameters())
    drop = B.Dropout(0.25, seed=5).to(DEV)
    flat = rand(1000, dtype=torch.float32, seed=2)
    first, second = drop(flat), drop(flat)
    assert torch.equal(first, B.dropout_forward(flat, 0.25, 5, 0)) and torch.equal(second, B.dropout_forward(flat, 0.25, 5, 1))
    other = B.Dropout(0.25)
    other.load_state_dict(drop.state_dict())
    assert torch.equal(other(flat), B.dropout_forward(flat, 0.25, 5, 2))
    assert drop.eval()(flat) is flat
    with pytest.raises(ValueError):
        B.GatedFFN(8, 8, activation="tanh")
    with pytest.raises(ValueError):
        B.GatedRefiner(16).to(DEV)(rand(4, 15, dtype=torch.float32, seed=1))


def test_a_new_refiner_leaves_the_frame_as_it_was():
    """Its blocks add zero, and the MLP rounds its features to the refiner's type in any case."""
    from nest_splat import blocks, renderer
    from nest_splat.mlp import NestMLP
    from nest_splat.scene import get_spec, make_scene
    sc = make_scene(get_spec("cfg1"))
    pc, ingp = renderer.scene_to_device(sc, DEV)
    bg = torch.zeros(3, device=DEV)
    ingp.mlp_rgb = NestMLP(sc.spec.C, 64, "f16").to(DEV)
    want = renderer.render(sc.cameras[0], pc, renderer.Pipe(), bg, ingp=ingp, with_surface=False)
    ingp.refiner = blocks.GatedRefiner(sc.spec.C, depth=2, dtype="f16").to(DEV).eval()
    got = renderer.render(sc.cameras[0], pc, renderer.Pipe(), bg, ingp=ingp, with_surface=False)
    assert torch.equal(got["features"], want["features"]) and torch.equal(got["render"], want["render"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_training_a_refiner(dtype):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_refiner.py")
    spec = importlib.util.spec_from_file_location("train_refiner", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    refiner, before, after = m.train(steps=60, dtype=dtype, device=str(DEV), log=lambda s: None)
    assert after < 0.9 * before
    assert all(torch.isfinite(p).all() for p in refiner.parameters())


# ---- offsets past 32 bits, float32 values that are not finite ----

def test_rows_past_4_gib(B):
    """The last rows of arrays over 4 GiB come out as the same rows by themselves: a row's result does not depend on its place."""
    for dtype, rows in ((torch.bfloat16, 34_000_003), (torch.float32, 17_000_003)):
        ws = ffn_case(1, 64, 96, 64, dtype)[1:4]
        x, dy = torch.zeros(rows, 64, dtype=dtype, device=DEV), torch.zeros(rows, 64, dtype=dtype, device=DEV)
        assert x.numel() * x.element_size() > 1 << 32
        x[-200:], dy[-200:] = rand(200, 64, dtype=dtype, seed=1), rand(200, 64, dtype=dtype, seed=2)
        tail = x[-200:].clone(), dy[-200:].clone()
        w = rand(64, dtype=dtype, seed=3)
        y, mean, rstd = B.layer_norm_forward(x, w)
        want = B.layer_norm_forward(tail[0], w)
        assert torch.equal(y[-200:], want[0])
        assert torch.equal(B.layer_norm_backward(dy, x, w, mean, rstd)[0][-200:], B.layer_norm_backward(tail[1], tail[0], w, *want[1:])[0])
        del y, mean, rstd
        assert torch.equal(B.gated_ffn_forward(x, *ws)[0][-200:], B.gated_ffn_forward(tail[0], *ws)[0])
        dx = B.gated_ffn_backward(dy, x, *ws)
        alone = B.gated_ffn_backward(tail[1], tail[0], *ws)
        assert torch.equal(dx[0][-200:], alone[0])
        for d, a in zip(dx[1:], alone[1:]):  # rows of zeros add nothing: the sums differ by their order alone
            assert torch.allclose(d.float(), a.float(), rtol=0, atol=float(a.float().abs().max()) * (2e-5 if dtype == torch.float32 else 2e-2))
        del x, dy, dx
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows", [4, 150])
def test_ffn_values_that_are_not_finite_stay_in_their_rows(B, rows, dtype):
    x, wg, wu, wd, dy = ffn_case(rows, 72, 200, 72, dtype)
    clean, cx = B.gated_ffn_forward(x, wg, wu, wd)[0], B.gated_ffn_backward(dy, x, wg, wu, wd)[0]
    x[1, 3], x[3, 71] = float("nan"), float("inf")
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[[1, 3]] = False
    y, dx = B.gated_ffn_forward(x, wg, wu, wd)[0], B.gated_ffn_backward(dy, x, wg, wu, wd)[0]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cx[keep])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any()


def test_ffn_float32_over_its_range(B):
    """Values from 2^-60 to 2^60 in one product: each is cut into parts by itself, the largest does not overflow."""
    x, wg, wu, wd, dy = ffn_case(100, 64, 96, 64, torch.float32)
    scale = torch.exp2(torch.arange(100, device=DEV, dtype=torch.float32).fmod(21) - 10)[:, None]
    ffn_check(B, x * scale, wg, wu, wd, dy, "relu")
    big = torch.full((70, 64), 2.0 ** 60, device=DEV)
    y = B.gated_ffn_forward(big, wg * 2.0 ** -60, wu * 2.0 ** -60, wd, "relu")[0]
    R.check(y, *R.ffn(big, wg * 2.0 ** -60, wu * 2.0 ** -60, wd, "relu")["y"], "y of 2^60")
