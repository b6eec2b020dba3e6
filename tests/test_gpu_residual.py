"""The residual block's operators (nest_splat.residual) against the formulas in
64 bits: values and gradients within the element-wise bounds of
residual_ref.py, at the sizes, layouts and values where they can go wrong."""
import pytest
import torch

import residual_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope="module")
def B():
    from nest_splat import residual
    return residual


def rand(*shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)


# ---- rows in 8 bits ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (7, 16), (5, 31), (4, 32), (9, 33), (1030, 64), (3, 47), (2, 100), (1, 4096), (300, 515)])
def test_pack8_is_the_definition(B, rows, cols, dtype):
    spread = torch.exp2(torch.randint(-9, 10, (rows, 1), generator=torch.Generator().manual_seed(rows)).float()).to(DEV)
    x = (rand(rows, cols, dtype=torch.float32, seed=cols) * spread).to(dtype)
    p = B.pack8(x)
    codes, steps, values = R.pack(x)
    assert p.codes.dtype == torch.int8 and torch.equal(p.codes, codes) and torch.equal(p.steps, steps)
    assert torch.equal(B.unpack8(p), values)
    assert p.nbytes == rows * (cols + -(-cols // 32))


@pytest.mark.parametrize("dtype", TYPES)
def test_pack8_ends_of_the_types_and_values_that_are_not_finite(B, dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(8, 70, dtype=dtype, device=DEV)
    x[0, 3], x[0, 40] = info.max, -info.max
    x[1, :32] = torch.arange(32, device=DEV).to(dtype) * info.tiny / 8
    x[2, 5], x[2, 33], x[3, 69] = float("inf"), float("nan"), float("-inf")
    x[4, :] = 0.5 - 2.0 ** -9   # 127.5 steps and its neighbours: the largest do not fit
    x[4, 1], x[4, 2], x[4, 3] = -(0.5 - 2.0 ** -9), 0.496, 0.25
    x[5, ::2] = -0.0
    codes, steps, values = R.pack(x)
    p = B.pack8(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.steps, steps)
    back = B.unpack8(p)
    assert torch.equal(back.isnan(), values.isnan()) and torch.equal(back.nan_to_num(0.0), values.nan_to_num(0.0))
    assert back[2, :64].isnan().all() and back[3, 64:].isnan().all() and not back[3, :64].isnan().any() and not back[2, 64:].isnan().any()


def test_pack8_no_rows_strides_and_alignment(B):
    assert B.unpack8(B.pack8(torch.zeros(0, 40, dtype=torch.float16, device=DEV))).shape == (0, 40)
    wide = rand(6, 10, 24, dtype=torch.bfloat16, seed=1).permute(2, 0, 1)
    for x in (wide, rand(1 + 7 * 24, dtype=torch.bfloat16, seed=2)[1:].view(7, 24), rand(9, 50, dtype=torch.bfloat16, seed=3)[:, 3:40]):
        assert torch.equal(B.unpack8(B.pack8(x)), R.pack(x.contiguous())[2])


# ---- dense layer ----

SIZES = [(1, 1, 1), (1, 2048, 512), (3, 70, 33), (4, 64, 200), (8, 515, 77), (16, 130, 64), (17, 64, 64), (33, 515, 130), (70, 7, 9),
         (257, 128, 48), (300, 96, 128), (1030, 16, 16), (64, 1024, 40), (100, 40, 1500), (513, 2048, 72)]


def linear_case(rows, cols, out, dtype, bias=True, residual=True, seed=1):
    return (rand(rows, cols, dtype=dtype, seed=seed), rand(out, cols, dtype=dtype, seed=seed + 1, scale=cols ** -0.5),
            rand(out, dtype=dtype, seed=seed + 2, scale=0.3) if bias else None,
            rand(rows, out, dtype=dtype, seed=seed + 3) if residual else None, rand(rows, out, dtype=dtype, seed=seed + 4))


def linear_check(B, x, w, b, r, dy, act, save8=False):
    flat = lambda t: None if t is None else t.reshape(-1, t.shape[-1])
    y, kept = B.linear_forward(x, w, b, act, r, training=True, save8=save8)
    packed = R.pack(x)[2] if save8 else None
    dx, dw, db = B.linear_backward(dy, B.pack8(x) if save8 else x, w, kept, act, with_bias=b is not None)
    ref = R.linear(flat(x), w, b, act, flat(r), flat(dy), save8, flat(packed))
    assert (db is None) == (b is None) and (kept is None) == (act is None)
    assert dx.shape == x.shape and y.shape == dy.shape
    for k, v in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        if v is not None:
            assert v.dtype == x.dtype
            R.check(v.reshape(ref[k][0].shape), *ref[k], f"{k} of {tuple(x.shape)} -> {w.shape[0]} {x.dtype} {act} save8={save8}")
    assert torch.equal(B.linear_forward(x, w, b, act, r)[0], y)   # what is kept does not change y
    return y, kept


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,out", SIZES)
def test_linear_values_and_gradients(B, rows, cols, out, dtype):
    linear_check(B, *linear_case(rows, cols, out, dtype), "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("rows,cols,out", [(5, 33, 40), (65, 48, 96), (200, 31, 17)])
def test_linear_activations_bias_and_residual(B, rows, cols, out, bias, residual, act, dtype):
    linear_check(B, *linear_case(rows, cols, out, dtype, bias, residual), act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("rows,cols,out", [(3, 40, 40), (130, 64, 128), (75, 515, 33), (1030, 32, 24)])
def test_linear_from_8_bits(B, rows, cols, out, act, dtype):
    linear_check(B, *linear_case(rows, cols, out, dtype), act, save8=True)


@pytest.mark.parametrize("cols,out", [(1, 1), (16, 16), (1, 64), (64, 1), (17, 33), (33, 50), (50, 33), (64, 64), (20, 40), (48, 17), (47, 48), (30, 63)])
@pytest.mark.parametrize("rows,act,save8", [(1, "silu", False), (70, "gelu", True), (70, "relu", False), (4111, "silu", True), (4111, None, False)])
def test_linear_narrow_float32(B, rows, cols, out, act, save8):
    linear_check(B, *linear_case(rows, cols, out, torch.float32, residual=rows != 1), act=act, save8=save8)


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_linear_kept_slopes_are_the_nearest_codes(B, act, dtype, save8):
    x, w, b, _, _ = linear_case(130, 72, 100 if save8 else 140, dtype)
    x[::3] *= 6
    _, kept = B.linear_forward(x, w, b, act, training=True, save8=save8)
    z, e_z = R.pre_activation(x, w, b)
    _, s, curve = R.act(z, act)
    if act == "relu":
        sure = z.abs() > e_z
        assert kept.dtype == torch.uint8 and torch.equal(kept.double()[sure], (26 + 200 * s)[sure])
        return
    e_s = curve * e_z + R.CALC * (1 + z.abs()) + 4 * R.F32
    step = R.slope_step(dtype, act, save8)
    if step == 0:
        assert kept.dtype == torch.float32 and ((kept.double() - s).abs() <= e_s).all()
        return
    assert kept.dtype == (torch.uint8 if step == 1 / R.COARSE else torch.int16)
    codes = kept.double() - (26 if step == 1 / R.COARSE else 0)
    assert ((codes - s / step).abs() <= 0.5 + e_s / step).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "silu"])
def test_linear_no_rows(B, dtype, act):
    x, w, b, r, dy = linear_case(0, 24, 40, dtype)
    y, kept = B.linear_forward(x, w, b, act, r, training=True)
    dx, dw, db = B.linear_backward(dy, x, w, kept, act)
    assert y.shape == (0, 40) and dx.shape == (0, 24) and not dw.any() and not db.any()


def test_linear_strides_leading_dimensions_and_alignment(B):
    _, w, b, r, dy = linear_case(60, 24, 40, torch.float16)
    w = rand(24, 40, dtype=torch.float16, seed=5, scale=0.2).t()
    x = rand(24, 6, 10, dtype=torch.float16, seed=7).permute(1, 2, 0)
    linear_check(B, x, w, b, r.view(6, 10, 40), dy.view(10, 6, 40).transpose(0, 1), "silu")
    flat = rand(1 + 60 * 24, dtype=torch.float16, seed=9)
    linear_check(B, flat[1:].view(60, 24), w, rand(41, dtype=torch.float16, seed=3)[1:], rand(60, 50, dtype=torch.float16, seed=6)[:, 5:45], dy, "gelu")


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("cols", [16, 33, 64, 70, 96, 128])
@pytest.mark.parametrize("out", [1, 32, 48, 64, 90, 128])
def test_linear_narrow_widths(B, cols, out, dtype):
    for rows, act in ((333, "silu"), (130, None)):
        linear_check(B, *linear_case(rows, cols, out, dtype), act)
        linear_check(B, *linear_case(rows, cols, out, dtype, residual=False), act, save8=True)
    x, w, b, r, dy = linear_case(70, cols, out, dtype)
    _, kept = B.linear_forward(x, w, b, "gelu", training=True, save8=True)
    got = B.linear_backward(dy, x, w, kept, "gelu")   # the slopes alone in 8 bits
    ref = R.linear(x, w, b, "gelu", None, dy, True)
    for k, v in zip(("dx", "dw", "db"), got):
        R.check(v, *ref[k], k)


def test_linear_narrow_many_turns(B):
    """More rows than the workgroups that run at once take in one turn, the last turn partial."""
    for rows, cols, out in ((256 * 3 * 128 + 77, 16, 32), (256 * 2 * 128 * 2 + 5, 64, 64), (256 * 64 * 2 + 31, 128, 128)):
        x, w, b, r, dy = linear_case(rows, cols, out, torch.bfloat16)
        linear_check(B, x, w, b, r, dy, "gelu")
        linear_check(B, x, w, b, r, dy, "gelu", save8=True)


def test_linear_gradients_that_are_not_wanted(B):
    for out in (40, 140):
        x, w, b, r, dy = linear_case(50, 24, out, torch.bfloat16)
        _, kept = B.linear_forward(x, w, b, "silu", r, training=True)
        want = B.linear_backward(dy, x, w, kept, "silu")
        for needs in ((True, False), (False, True), (False, False)):
            for bias in (True, False):
                got = B.linear_backward(dy, x, w, kept, "silu", with_bias=bias, needs=needs)
                for g, v, n in zip(got, want, (*needs, bias)):
                    assert torch.equal(g, v) if n else g is None


@pytest.mark.parametrize("out", [40, 140])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_without_x(B, dtype, out):
    """dx and dbias alone need no x where slopes are kept, or there are none."""
    x, w, b, r, dy = linear_case(50, 24, out, dtype)
    for act, save8 in ((None, False), ("silu", True), ("relu", True)):
        _, kept = B.linear_forward(x, w, b, act, r, training=True, save8=save8)
        want = B.linear_backward(dy, x, w, kept, act)
        dx, dw, db = B.linear_backward(dy, None, w, kept, act, needs=(True, False))
        assert torch.equal(dx, want[0]) and dw is None and torch.equal(db, want[2])
    for act in (None, "gelu"):
        for save8 in (False, True):
            ps = [t.clone().requires_grad_(k in (0, 2)) for k, t in enumerate((x, w, b))]
            got = torch.autograd.grad(B.linear(*ps, act, save8=save8), (ps[0], ps[2]), dy)
            _, kept = B.linear_forward(x, w, b, act, training=True, save8=save8)
            want = B.linear_backward(dy, x, w, kept, act)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_linear_values_that_are_not_finite_stay_in_their_rows(B, dtype):
    for rows in (9, 100):
        x, w, b, r, dy = linear_case(rows, 40, 24, dtype)
        w = w.abs() + 0.1
        clean, _ = B.linear_forward(x, w, b, "relu", r)
        x[2, 5], x[7, 39], x[5, 0] = float("nan"), float("inf"), float("-inf")
        y, kept = B.linear_forward(x, w, b, "relu", r, training=True)
        rest = torch.ones(rows, dtype=torch.bool, device=DEV)
        rest[[2, 5, 7]] = False
        assert torch.equal(y[rest], clean[rest])
        assert y[2].isnan().all() and (y[7] == float("inf")).all() and torch.equal(y[5], r[5])
        for save8 in (False, True):
            z, kept = B.linear_forward(x, w, b, "silu", training=True, save8=save8)
            assert z[2].isnan().all() and (not save8 or (kept[2] == 255).all())
            dx = B.linear_backward(dy, x, w, kept, "silu", needs=(True, False))[0]
            assert dx[2].isnan().all() and not dx[rest].isnan().any()
        _, kept = B.linear_forward(x, w, b, "relu", training=True)
        dx = B.linear_backward(dy, x, w, kept, "relu", needs=(True, False))[0]
        assert dx[7].isfinite().all() and not dx[5].any()   # slopes 1 and 0


def test_linear_repeats_bit_for_bit_and_autograd(B):
    x, w, b, r, dy = linear_case(3000, 96, 160, torch.bfloat16)
    y, kept = B.linear_forward(x, w, b, "gelu", r, training=True)
    first = B.linear_backward(dy, x, w, kept, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(first, B.linear_backward(dy, x, w, kept, "gelu")))
    ps = [t.clone().requires_grad_() for t in (x, w, b, r)]
    out = B.linear(ps[0], ps[1], ps[2], "gelu", ps[3])
    assert torch.equal(out, y)
    got = torch.autograd.grad(out, ps, dy)
    assert all(torch.equal(p, q) for p, q in zip((*first, dy), got))
    _, k8 = B.linear_forward(x, w, b, "gelu", r, training=True, save8=True)
    want = B.linear_backward(dy, B.pack8(x), w, k8, "gelu")
    got = torch.autograd.grad(B.linear(ps[0], ps[1], ps[2], "gelu", ps[3], save8=True), ps, dy)
    assert all(torch.equal(p, q) for p, q in zip((*want, dy), got))


# ---- the residual stream between two norms ----

def norm_case(rows, cols, dtype, pdt=None, gates=1, seed=1):
    pdt = pdt or dtype
    one = lambda k: rand(cols, dtype=pdt, seed=seed + k, scale=0.2, shift=1.0)
    return dict(x=rand(rows, cols, dtype=dtype, seed=seed, shift=0.3), h=rand(rows, cols, dtype=dtype, seed=seed + 1, scale=2.0),
                gate=rand(gates, cols, dtype=pdt, seed=seed + 2, shift=0.5) if gates else None, post=one(3), pre=one(4),
                dr=rand(rows, cols, dtype=dtype, seed=seed + 5), dy=rand(rows, cols, dtype=dtype, seed=seed + 6))


def norm_check(B, c, scale=1.0, eps=1e-6, what=""):
    x, h, gate, post, pre = (c[k] for k in ("x", "h", "gate", "post", "pre"))
    D = x.shape[-1]
    flat = lambda t: None if t is None else t.reshape(-1, D)
    r, y, stats = B.residual_norm_forward(x, h, gate, post, pre, scale, eps)
    what = f"{what} of {tuple(x.shape)} {x.dtype}, gate {None if gate is None else tuple(gate.shape)}"
    if h is None:
        assert torch.equal(r, x)
    else:
        R.check(flat(r), *R.residual_norm_r(flat(x), flat(h), flat(gate), post, scale, eps), "r" + what)
    if pre is None:
        assert y is None
    else:
        R.check(flat(y), *R.residual_norm_y(flat(r), pre, eps), "y" + what)
    got = dict(zip(("dx", "dh", "dgate", "dpost", "dpre"), B.residual_norm_backward(c["dr"], c["dy"], r, h, gate, post, pre, stats, scale)))
    ref = R.residual_norm_back(flat(c["dr"]), flat(c["dy"]), flat(r), flat(h), flat(gate), post, pre, scale, eps)
    for k, v in got.items():
        assert (v is None) == (k not in ref), k
        if v is not None:
            assert v.dtype == (x.dtype if k in ("dx", "dh") else next(t.dtype for t in (post, pre, gate) if t is not None))
            R.check(v.reshape(ref[k][0].shape), *ref[k], k + what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 2048), (70, 7), (513, 64), (37, 129), (1030, 16), (9, 515), (5, 1024), (6, 1031),
                                       (3, 2049), (2, 4100), (3, 8192), (2, 8191), (700, 520)])
def test_residual_norm_values_and_gradients(B, rows, cols, dtype):
    norm_check(B, norm_case(rows, cols, dtype), scale=0.75)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,gates", [(12, 40, 3), (12, 40, 12), (600, 64, 2), (600, 64, 300), (600, 64, 600), (4000, 16, 1000), (6, 1500, 2),
                                             (6, 1500, 6), (6, 5000, 6), (40, 5000, 5), (7, 700, 7), (3000, 8, 1)])
def test_residual_norm_gates(B, rows, cols, gates, dtype):
    norm_check(B, norm_case(rows, cols, dtype, gates=gates))


@pytest.mark.parametrize("rows,cols,gates", [(9000, 24, 3000), (6000, 1500, 3000), (5000, 4100, 2500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_residual_norm_more_gates_than_workgroups(B, rows, cols, gates, dtype):
    norm_check(B, norm_case(rows, cols, dtype, gates=gates))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(41, 200), (6, 1300)])
def test_residual_norm_parts_that_are_left_out(B, rows, cols, dtype):
    full = norm_case(rows, cols, dtype)
    for drop in (("gate",), ("post",), ("pre", "dy"), ("gate", "post"), ("gate", "pre", "dy"), ("post", "pre", "dy"), ("gate", "post", "pre", "dy"),
                 ("dr",), ("dy",), ("h", "gate", "post"), ("h", "gate", "post", "dr"), ("h", "gate", "post", "dy")):
        norm_check(B, {k: None if k in drop else v for k, v in full.items()}, what=f" without {drop}")
    many = norm_case(rows * 2, cols, dtype, gates=2)
    for drop in (("post",), ("pre", "dy"), ("dr",)):
        norm_check(B, {k: None if k in drop else v for k, v in many.items()}, what=f" without {drop}")
    each = norm_case(rows, cols, dtype, gates=rows)
    for drop in (("post",), ("pre", "dy"), ("dr",), ("post", "pre", "dy")):
        norm_check(B, {k: None if k in drop else v for k, v in each.items()}, what=f" without {drop}")


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("gates", [0, 1, 4, 24])
def test_residual_norm_float32_parameters(B, dtype, gates):
    for cols in (72, 1100, 8192):
        norm_check(B, norm_case(24, cols, dtype, torch.float32, gates=gates))


def test_residual_norm_zero_rows_large_values_and_other_eps(B):
    c = norm_case(8, 96, torch.float32)
    c["h"][0] = 0.0
    c["x"][1], c["h"][1] = 0.0, 0.0
    c["x"][2] *= 1000.0
    norm_check(B, c)
    norm_check(B, c, eps=0.1, scale=-2.0)


def test_residual_norm_nan_and_infinity_stay_in_their_rows(B):
    c = norm_case(9, 130, torch.float32)
    args = [c[k] for k in ("x", "h", "gate", "post", "pre")]
    clean = B.residual_norm_forward(*args)
    c["x"][2, 5], c["h"][7, 129] = float("nan"), float("inf")
    r, y, stats = B.residual_norm_forward(*args)
    rest = torch.ones(9, dtype=torch.bool, device=DEV)
    rest[[2, 7]] = False
    assert torch.equal(y[rest], clean[1][rest]) and torch.equal(r[rest], clean[0][rest])
    assert y[2].isnan().all() and y[7].isnan().all()
    back = B.residual_norm_backward(c["dr"], c["dy"], clean[0], args[1], *args[2:], clean[2])
    got = B.residual_norm_backward(c["dr"], c["dy"], r, args[1], *args[2:], stats)
    assert all(torch.equal(p[rest], q[rest]) for p, q in zip(got[:2], back[:2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gates", [0, 1, 3])
def test_residual_norm_no_rows(B, dtype, gates):
    c = norm_case(0, 33, dtype, gates=gates)
    r, y, stats = B.residual_norm_forward(c["x"], c["h"], c["gate"] if gates < 2 else None, c["post"], c["pre"])
    assert r.shape == y.shape == (0, 33)
    back = B.residual_norm_backward(c["dr"], c["dy"], r, c["h"], c["gate"] if gates < 2 else None, c["post"], c["pre"], stats)
    assert back[0].shape == (0, 33) and not any(t.any() for t in back if t is not None)


def test_residual_norm_strides_leading_dimensions_and_alignment(B):
    c = norm_case(60, 24, torch.float16)
    c["x"] = rand(24, 6, 10, dtype=torch.float16, seed=7).permute(1, 2, 0)
    for k in ("h", "dr", "dy"):
        c[k] = c[k].view(10, 6, 24).transpose(0, 1)
    for shape in ((24,), (6, 24), (6, 1, 24), (6, 10, 24), (1, 1, 24)):
        c["gate"] = rand(*shape, dtype=torch.float16, seed=8)
        norm_check(B, c)
    c = norm_case(7, 24, torch.float16)
    c["x"] = rand(1 + 7 * 24, dtype=torch.float16, seed=9)[1:].view(7, 24)
    c["dy"] = rand(7, 30, dtype=torch.float16, seed=10)[:, 3:27]
    norm_check(B, c)


def test_residual_norm_repeats_bit_for_bit_and_autograd(B):
    for gates in (1, 5, 5000):
        c = norm_case(5000, 96, torch.bfloat16, gates=gates)
        ins = [c[k] for k in ("x", "h", "gate", "post", "pre")]
        r, y, stats = B.residual_norm_forward(*ins, 0.5)
        first = B.residual_norm_backward(c["dr"], c["dy"], r, *ins[1:], stats, 0.5)
        again = B.residual_norm_backward(c["dr"], c["dy"], r, *ins[1:], stats, 0.5)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        ps = [t.clone().requires_grad_() for t in ins]
        out = B.residual_norm(*ps, scale=0.5)
        assert torch.equal(out[0], r) and torch.equal(out[1], y)
        assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(out, ps, (c["dr"], c["dy"]))))
        only = torch.autograd.grad(B.residual_norm(*ps, scale=0.5)[1], ps[:2], c["dy"])
        want = B.residual_norm_backward(None, c["dy"], r, *ins[1:], stats, 0.5)
        assert all(torch.equal(p, q) for p, q in zip(want, only))
    x, pre = ps[0], ps[4]
    r, y = B.residual_norm(x, pre=pre)
    assert r is x
    dx, dpre = torch.autograd.grad((r, y), (x, pre), (c["dr"], c["dy"]))
    back = B.residual_norm_backward(None, c["dy"], ins[0], pre=ins[4], stats=B.residual_norm_forward(ins[0], pre=ins[4])[2])
    assert torch.equal(dx, (c["dr"] + back[0])) and torch.equal(dpre, back[4])


# ---- embedding ----

def embed_check(B, ids, table, scale=1.25, residual=None, dy=None):
    y = B.embedding_forward(ids, table, scale, residual)
    D = table.shape[1]
    assert y.shape == ids.shape + (D,) and y.dtype == table.dtype
    R.check(y.reshape(-1, D), *R.embedding(ids, table, scale, residual), f"y of {tuple(ids.shape)}, table {tuple(table.shape)} {table.dtype}")
    if dy is not None:
        got = B.embedding_backward(dy, ids, table.shape[0], scale)
        assert got.dtype == dy.dtype
        R.check(got, *R.embedding_back(dy, ids, table.shape[0], scale), f"dtable of {tuple(ids.shape)}, table {tuple(table.shape)} {table.dtype}")
        assert torch.equal(got, B.embedding_backward(dy, ids, table.shape[0], scale))


def some_ids(n, rows, seed, skew=1, outside=True, dtype=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lo, hi = (-1, rows + 1) if outside else (0, rows)
    u = torch.rand(n, generator=g, device=DEV) ** skew
    return (lo + u * (hi - lo)).long().clamp(max=hi - 1).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,cols,skew", [(1, 1, 1, 1), (1, 5, 64, 1), (15, 3, 7, 1), (16, 1, 64, 1), (17, 300, 33, 1), (33, 2, 8, 1), (100, 255, 130, 1),
                                              (1000, 256, 64, 1), (1000, 257, 20, 4), (5000, 70000, 24, 3), (5000, 1, 16, 1), (4096, 40, 515, 2),
                                              (300, 50, 2048, 1), (20000, 3, 64, 6), (65, 9, 1100, 1), (70000, 300, 32, 1), (8192, 5000, 40, 2),
                                              (8193, 5000, 40, 2), (70001, 1024, 64, 1), (3001, 1025, 64, 1), (9000, 384, 128, 1), (9000, 385, 128, 1),
                                              (600, 4096, 9, 1), (130000, 200, 96, 1), (12000, 7, 4096, 3)])
def test_embedding_values_and_gradients(B, n, rows, cols, skew, dtype):
    ids = some_ids(n, rows, seed=n, skew=skew)
    embed_check(B, ids, rand(rows, cols, dtype=dtype, seed=1), 1.25, rand(n, cols, dtype=dtype, seed=2), rand(n, cols, dtype=dtype, seed=3))


def test_embedding_runs_that_end_at_chunks(B):
    """Sorted ids whose runs begin and end at, before and after multiples of the chunks that the gradient sums, past the sizes
    whose positions are sorted at once too."""
    for lengths in ([16] * 40, [32, 16, 48, 64, 1, 15], [17, 15, 31, 33, 1, 1, 1, 13], [1] * 200, [640], [5, 2000, 5], [1024, 1024, 1023, 1025], [16, 5000, 16], [9000], [1, 20000, 1, 300, 5], [2048] * 9):
        ids = torch.cat([torch.full((k,), 3 * i + 1, device=DEV) for i, k in enumerate(lengths)])
        rows = 3 * len(lengths) + 2
        embed_check(B, ids, rand(rows, 72, dtype=torch.float32, seed=4), 1.0, None, rand(len(ids), 72, dtype=torch.float32, seed=5))
        mixed = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1)).to(DEV)]
        embed_check(B, mixed, rand(rows, 72, dtype=torch.float32, seed=4), 1.0, None, rand(len(ids), 72, dtype=torch.float32, seed=6))


def test_embedding_ids_of_both_types_outside_and_extreme(B):
    table, dy = rand(50, 40, dtype=torch.bfloat16, seed=1), rand(300, 40, dtype=torch.bfloat16, seed=2)
    for dtype in (torch.int32, torch.int64):
        ids = some_ids(300, 50, seed=4, dtype=dtype)
        info = torch.iinfo(dtype)
        ids[:6] = torch.tensor([info.max, info.min, -1, 50, 51, 49], dtype=dtype)
        embed_check(B, ids, table, 0.5, None, dy)
        embed_check(B, ids.view(3, 100), table, 0.5, rand(3, 100, 40, dtype=torch.bfloat16, seed=6), dy.view(3, 100, 40))
    none = torch.full((300,), -1, device=DEV)
    r = rand(300, 40, dtype=torch.bfloat16, seed=6)
    r[3, 4] = float("nan")
    y = B.embedding_forward(none, torch.full_like(table, float("nan")), 0.5, r)
    assert torch.equal(y.nan_to_num(7.0), r.nan_to_num(7.0)) and not B.embedding_forward(none, table).any()
    assert not B.embedding_backward(dy, none, 50).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_no_rows_strides_and_alignment(B, dtype):
    table = rand(9, 24, dtype=dtype, seed=1)
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    assert B.embedding_forward(empty, table).shape == (0, 24)
    assert not B.embedding_backward(torch.empty(0, 24, dtype=dtype, device=DEV), empty, 9).any()
    ids = some_ids(14, 9, seed=2, outside=False)
    embed_check(B, ids[::2], rand(24, 9, dtype=dtype, seed=3).t(), 1.0, rand(7, 30, dtype=dtype, seed=4)[:, 2:26], rand(7, 30, dtype=dtype, seed=5)[:, 1:25])
    embed_check(B, ids, rand(1 + 9 * 24, dtype=dtype, seed=6)[1:].view(9, 24), -1.0, None, rand(1 + 14 * 24, dtype=dtype, seed=7)[1:].view(14, 24))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [20, 3000])
def test_embedding_infinities_and_nan_of_dy_stay_with_their_ids(B, rows, dtype):
    n, inf, nan = 700, float("inf"), float("nan")
    ids = some_ids(n, rows, seed=1, outside=False)
    ids[:12] = torch.arange(12, device=DEV)
    dy = rand(n, 48, dtype=dtype, seed=4)
    dy[0, 3], dy[1, 4], dy[2, 5] = inf, -inf, nan
    dy[3, 6], dy[4, 7] = inf, torch.finfo(dtype).max
    ids[600] = 3
    dy[600, 6] = -inf   # with the infinity above: NaN
    ids[601], dy[601, 8] = -1, nan   # of no id
    clean = R.embedding_back(dy, ids, rows, -2.0)[0]
    got = B.embedding_backward(dy, ids, rows, -2.0)
    assert torch.equal(got.isnan(), clean.isnan()) and torch.equal(got.isinf(), clean.to(dtype).isinf())
    assert got[0, 3] == -inf and got[1, 4] == inf and got[2, 5].isnan() and got[3, 6].isnan()
    finite = clean.to(dtype).isfinite()
    value, bound = R.embedding_back(torch.where(dy.isfinite(), dy, torch.zeros_like(dy)), ids, rows, -2.0)
    assert ((got.double() - value).abs() <= bound)[finite].all()
    assert torch.equal(got, B.embedding_backward(dy, ids, rows, -2.0)) or got.isnan().any()


def test_embedding_nan_stays_in_its_row_and_autograd(B):
    ids = some_ids(500, 20, seed=1, outside=False)
    table, r, dy = rand(20, 48, dtype=torch.float16, seed=2), rand(500, 48, dtype=torch.float16, seed=3), rand(500, 48, dtype=torch.float16, seed=4)
    bad = dy.clone()
    bad[100] = float("nan")
    got, clean = B.embedding_backward(bad, ids, 20), B.embedding_backward(dy, ids, 20)
    rest = torch.arange(20, device=DEV) != ids[100]
    assert got[ids[100]].isnan().all() and torch.equal(got[rest], clean[rest])
    ps = [t.clone().requires_grad_() for t in (table, r)]
    out = B.embedding(ids, ps[0], 0.75, ps[1])
    assert torch.equal(out, B.embedding_forward(ids, table, 0.75, r))
    dt, dres = torch.autograd.grad(out, ps, dy)
    assert torch.equal(dt, B.embedding_backward(dy, ids, 20, 0.75)) and torch.equal(dres, dy)


# ---- gradients against differences ----

def test_gradients_are_the_slopes_of_the_values(B):
    """Directional differences of a float32 loss over the operators as they compute it, extrapolated from two steps: what the
    extrapolation leaves is below what the two steps differ by, and the values' rounding adds 8 units of each over the step."""
    ids = some_ids(40, 6, seed=9)
    table = rand(6, 24, dtype=torch.float32, seed=10)
    x, w, b, r, dy = linear_case(40, 24, 24, torch.float32)
    c = norm_case(40, 24, torch.float32, gates=4)
    ins = [x, w, b, c["x"], c["gate"], c["post"], c["pre"], table]

    def values(x, w, b, s, gate, post, pre, table):
        h = B.linear(B.embedding(ids, table, 1.5, x), w, b, "gelu", x)
        return B.residual_norm(s, h, gate, post, pre, 0.8)

    def loss(ts):
        p, q = values(*ts)
        return float((p.double() * c["dr"].double()).sum() + (q.double() * c["dy"].double()).sum()), float((p.abs() * c["dr"].abs()).sum() + (q.abs() * c["dy"].abs()).sum())

    ps = [t.clone().requires_grad_() for t in ins]
    grads = torch.autograd.grad(values(*ps), ps, (c["dr"], c["dy"]))
    for k, g in enumerate(grads):
        way = rand(*ins[k].shape, dtype=torch.float32, seed=50 + k)
        slope = float((g.double() * way.double()).sum())
        found = []
        for step in (2.0 ** -5, 2.0 ** -6):
            ends = [loss([t + s * step * way if i == k else t for i, t in enumerate(ins)]) for s in (1, -1)]
            found.append((ends[0][0] - ends[1][0]) / (2 * step))
            noise = 8 * R.F32 * ends[0][1] / step
        best = (4 * found[1] - found[0]) / 3
        assert abs(best - slope) <= abs(found[0] - found[1]) + 2 * noise, (k, slope, found)
