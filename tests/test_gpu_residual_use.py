"""The residual block's operators as programs use them: together in a ViewRefiner and render(), under autograd, on streams, in
graphs, and past the sizes that 32 bits count."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import residual_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def B():
    from nest_splat import residual
    return residual


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def trained(B, C, views, seed=3, **kw):
    """A refiner whose every part changes its input."""
    r = B.ViewRefiner(C, views, **kw).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    with torch.no_grad():
        r.embed.weight.copy_(torch.randn(r.embed.weight.shape, generator=g, device=DEV) * 0.5)
        for p in [r.first, *r.joins.parameters(), *(q.bias for q in (*r.ups, *r.downs))]:
            p.copy_(p + torch.randn(p.shape, generator=g, device=DEV) * 0.3)
    return r


def plain_refiner(r, x, views):
    """The refiner's formula in 64 bits."""
    x = x.double()
    if views is not None:
        inside = (views >= 0) & (views < r.views)
        x = x + torch.where(inside[..., None], r.embed.weight.double()[views.clamp(0, r.views - 1).long()], 0.0)
    rms = lambda v: v * R.inv_rms(v, 1e-6)
    y = rms(x) * r.first.double()
    for up, down, join in zip(r.ups, r.downs, r.joins):
        h = y @ up.weight.double().T + up.bias.double()
        h = torch.nn.functional.gelu(h) @ down.weight.double().T + down.bias.double()
        x = x + rms(h) * join.post.double() * join.gate.double()
        y = None if join.pre is None else rms(x) * join.pre.double()
    return x


@pytest.mark.parametrize("features,hidden,depth", [(16, 32, 1), (64, 128, 2), (24, 200, 3)])
def test_refiner_is_its_formula_and_trains(B, features, hidden, depth):
    """In float32: each of a block's two products is off by gamma(length) of its terms' magnitudes, here at most 16 times the
    result's norm, each norm and join by a few units; depth blocks and the way back add up to 4 depth such steps."""
    r = trained(B, features, 5, hidden=hidden, depth=depth, dtype="f32")
    x = rand(300, features, seed=1)
    views = torch.randint(-1, 6, (300,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    dy = rand(300, features, seed=4)
    bound = 4 * depth * 16 * R.gamma(hidden + 300)
    x.requires_grad_()
    y = r(x, views)
    want = plain_refiner(r, x, views)
    assert y.dtype == x.dtype and float((y.detach().double() - want.detach()).norm() / want.detach().norm()) < bound
    ps = [x, *r.parameters()]
    got, ref = torch.autograd.grad(y, ps, dy), torch.autograd.grad(want, ps, dy.double())
    for p, g, w in zip(ps, got, ref):
        assert g.shape == p.shape and float((g.double() - w.double()).norm()) < bound * float(w.double().norm()), tuple(p.shape)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("save8", [False, True])
def test_refiner_in_16_bits(B, dtype, save8):
    """Against float32 of the same weights: the stream, and each of the operands between, are off by a rounding of the type, 8 of
    them a block; with 8 bits the weights' gradients are off by the codes, 2^-7 of a group's largest (within 4 of its root mean
    square), and the slopes by half a step of 1/200 on values of about 1/2."""
    r = trained(B, 48, 3, hidden=96, depth=2, dtype=dtype, save8=save8)
    full = copy.deepcopy(r)
    full.dtype = full.embed.dtype = torch.float32
    for q in (*full.ups, *full.downs):
        q.dtype, q.save8 = torch.float32, False
    x, views = rand(500, 48, seed=1), torch.randint(0, 3, (500,), device=DEV)
    unit = R.R.UNIT[r.dtype]
    bound = 16 * unit
    y = r(x, views)
    want = full(x, views)
    assert float((y - want).detach().norm() / want.detach().norm()) < bound
    slack = 2 * bound + (2.0 ** -7 * 4 + 0.01 if save8 else 0)
    for g, w in zip(torch.autograd.grad(y.square().sum(), list(r.parameters())), torch.autograd.grad(want.square().sum(), list(full.parameters()))):
        assert float((g - w).norm()) < slack * float(w.norm()), tuple(w.shape)


def test_refiner_arguments_and_a_new_one(B):
    r = B.ViewRefiner(16, 4, dtype="bf16").to(DEV)
    x = rand(70, 16, seed=1)
    assert torch.equal(r(x, 2), x.bfloat16().float()) and torch.equal(r(x), x.bfloat16().float())
    assert r(x[:0], 1).shape == (0, 16)
    for bad in (lambda: r(x, 4), lambda: r(x, -1), lambda: r(x[:, :8]), lambda: r(x, torch.zeros(69, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        r(x, torch.zeros(70, device=DEV))
    r = trained(B, 16, 4, dtype="f32")
    image = rand(16, 6, 9, seed=2)
    rows = image.reshape(16, -1).t()
    assert torch.equal(r.refine_image(image, 3), r(rows, torch.full((54,), 3, device=DEV)).t().reshape(16, 6, 9))
    assert torch.equal(r.refine_image(image), r(rows).t().reshape(16, 6, 9))


def test_render_decodes_through_the_view_of_the_camera(B):
    import dataclasses

    from nest_splat import renderer
    from nest_splat.scene import get_spec, make_scene
    sc = make_scene(get_spec("cfg1"))
    pc, ingp = renderer.scene_to_device(sc, DEV)
    bg, cam = torch.zeros(3, device=DEV), sc.cameras[0]
    frame = lambda c: renderer.render(c, pc, renderer.Pipe(), bg, ingp=ingp, with_surface=False)
    plain = frame(cam)
    ingp.refiner = trained(B, sc.spec.C, 3, dtype="f32").train()
    for view in (None, 0, 2):
        got = frame(dataclasses.replace(cam, view=view))
        assert not got["render"].requires_grad and ingp.refiner.training
        with torch.no_grad():
            refined = ingp.refiner.refine_image(plain["features"], view)
        want = ingp.mlp_rgb.decode_image(refined, renderer.view_ray_matrix(cam), alpha=plain["allmap"][1:2], bg=None)
        assert torch.equal(got["render"], want) and not torch.equal(want, plain["render"])
    with pytest.raises(ValueError):
        frame(dataclasses.replace(cam, view=3))


# ---- autograd ----

def test_nothing_is_kept_where_nothing_is_recorded(B):
    x, w, b = rand(4096, 256, seed=1, dtype=torch.bfloat16), rand(256, 256, seed=2, dtype=torch.bfloat16).requires_grad_(), rand(256, seed=3, dtype=torch.bfloat16)

    def peak(f):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        f()
        return torch.cuda.max_memory_allocated()

    with torch.no_grad():
        B.linear(x, w, b, "gelu")
        least = peak(lambda: B.linear(x, w.detach(), b, "gelu"))
        assert peak(lambda: B.linear(x, w, b, "gelu")) <= least
    assert peak(lambda: B.linear(x, w, b, "gelu")) >= least + 2 * 4096 * 256


def test_saved_in_8_bits_holds_less(B):
    x, w = rand(8192, 512, seed=1, dtype=torch.bfloat16), rand(512, 512, seed=2, dtype=torch.bfloat16).requires_grad_()
    held = []
    for save8 in (False, True):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = B.linear(x * 1, w, None, "silu", save8=save8)   # an x that the graph alone holds
        held.append(torch.cuda.memory_allocated() - before - y.nbytes)
        y.backward(torch.ones_like(y))
    n = 8192 * 512
    assert held[0] >= 4 * n and held[1] <= 2.1 * n + (1 << 20)


@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_forward(B, reentrant):
    r = trained(B, 32, 4, depth=2, dtype="f32", save8=True)
    x, views = rand(100, 32, seed=1).requires_grad_(), torch.randint(0, 4, (100,), device=DEV)
    want = torch.autograd.grad(r(x, views).square().sum(), [x, *r.parameters()])
    checkpoint(r, x, views, use_reentrant=reentrant).square().sum().backward()
    assert all(torch.equal(p, q) for p, q in zip(want, [x.grad, *(p.grad for p in r.parameters())]))


def test_broadcast_gradients_and_inputs_that_need_none(B):
    """dy as sum() gives it, of stride 0; each input alone needing a gradient."""
    x, w, b, r = (rand(*s, seed=k).requires_grad_() for k, s in enumerate(((40, 24), (140, 24), (140,), (40, 140))))
    want = torch.autograd.grad((B.linear(x, w, b, "silu", r) * torch.ones(40, 140, device=DEV)).sum(), (x, w, b, r))
    got = torch.autograd.grad(B.linear(x, w, b, "silu", r).sum(), (x, w, b, r))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    for k, t in enumerate((x, w, b, r)):
        args = [t if i == k else a.detach() for i, a in enumerate((x, w, b, r))]
        assert torch.equal(torch.autograd.grad(B.linear(args[0], args[1], args[2], "silu", args[3]).sum(), t)[0], want[k])
    s, h, g, post, pre = (rand(*s, seed=k).requires_grad_() for k, s in enumerate(((40, 24), (40, 24), (24,), (24,), (24,))))
    def loss(*a):
        p, q = B.residual_norm(*a, scale=0.5)
        return p.sum() + q.sum()
    want = torch.autograd.grad(loss(s, h, g, post, pre), (s, h, g, post, pre))
    for k, t in enumerate((s, h, g, post, pre)):
        args = [t if i == k else a.detach() for i, a in enumerate((s, h, g, post, pre))]
        assert torch.equal(torch.autograd.grad(loss(*args), t)[0], want[k])
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        gx = torch.autograd.grad(B.linear(x, w, b, "silu").square().sum(), x, create_graph=True)[0]
        torch.autograd.grad(gx.sum(), w)


def test_refusals(B):
    x, w, b, dy = rand(50, 24, dtype=torch.bfloat16, seed=1), rand(140, 24, dtype=torch.bfloat16, seed=2), rand(140, dtype=torch.bfloat16, seed=3), rand(50, 140, dtype=torch.bfloat16, seed=4)
    _, kept = B.linear_forward(x, w, b, "silu", training=True)
    narrow = w[:40].contiguous()
    _, again = B.linear_forward(x, narrow, b[:40], "silu", training=True)
    value = [lambda: B.linear_forward(x, w, b, "tanh"), lambda: B.linear_forward(x[:, :8], w), lambda: B.linear_forward(x, w, b[:9]),
             lambda: B.linear_forward(x, w, residual=dy[:9]), lambda: B.linear_forward(x, w[0]), lambda: B.linear_forward(x, w.cpu()),
             lambda: B.linear_backward(dy, x, w, None, "silu"), lambda: B.linear_backward(dy[:9], x, w, kept, "silu"),
             lambda: B.linear_backward(dy, x, w, kept[:9], "silu"), lambda: B.linear_backward(dy, x, w, kept.float(), "silu"),
             lambda: B.linear_backward(dy, x, w, b, "silu"), lambda: B.linear_backward(dy, None, w, kept, "silu"),
             lambda: B.linear_backward(dy, B.pack8(x.half()), w, kept, "silu"), lambda: B.linear_backward(dy, B.pack8(x[:9]), w, kept, "silu"),
             lambda: B.linear_backward(dy[:, :40], B.pack8(x), narrow, again, "silu"), lambda: B.linear_backward(dy[:, :40], None, narrow, again, "silu", needs=(True, False)),
             lambda: B.linear_backward(dy[:, :40], x, narrow, again[:9], "silu"), lambda: B.residual_norm_forward(x, x[:9]),
             lambda: B.residual_norm_forward(x, x, x[0, :9]), lambda: B.residual_norm_forward(x, x, x[:7]), lambda: B.residual_norm_forward(x.view(5, 10, 24), x.view(5, 10, 24), x[:10]),
             lambda: B.residual_norm_forward(x, x, pre=x[0, :9]), lambda: B.residual_norm_forward(x.new_zeros(2, 8193), x.new_zeros(2, 8193)),
             lambda: B.residual_norm_backward(x, x, x, x), lambda: B.residual_norm_backward(x, None, x, x), lambda: B.residual_norm_backward(x, None, x, x, stats=x),
             lambda: B.embedding_forward(torch.zeros(5, dtype=torch.int64, device=DEV), x[0]), lambda: B.embedding_forward(torch.zeros(5, dtype=torch.int64), x),
             lambda: B.embedding_forward(torch.zeros(5, dtype=torch.int64, device=DEV), x, residual=x), lambda: B.embedding_backward(x, torch.zeros(5, dtype=torch.int64, device=DEV), 3),
             lambda: B.embedding_backward(x, torch.zeros(50, dtype=torch.int64, device=DEV), 0), lambda: B.pack8(x[0, 0]),
             lambda: B.embedding_forward(torch.zeros(5, dtype=torch.int64, device=DEV), x[:0])]
    for k, call in enumerate(value):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {k} was taken")
    for k, call in enumerate((lambda: B.linear_forward(x, w.half()), lambda: B.linear_forward(x, w, b.float()), lambda: B.residual_norm_forward(x, x.half()),
                              lambda: B.residual_norm_forward(x, x, pre=x[0].half()), lambda: B.residual_norm_forward(x, x, post=x[0], pre=x[0].float()),
                              lambda: B.embedding_forward(torch.zeros(5, device=DEV), x), lambda: B.embedding_forward(torch.zeros(5, dtype=torch.int16, device=DEV), x))):
        with pytest.raises(TypeError):
            call()
            pytest.fail(f"call {k} was taken")


# ---- streams and graphs ----

def step(B, x, w, b, h, ids, table, dr, dy, out=24):
    """One forward and backward call of each operator: all results."""
    rows = B.embedding_forward(ids, table, 1.5, x)
    y, kept = B.linear_forward(rows, w, b, "gelu", training=True, save8=True)
    r, z, stats = B.residual_norm_forward(x, y[:, :24].contiguous(), None, table[0], table[1])
    back = B.residual_norm_backward(dr, dr, r, h, table[2], table[0], table[1], stats)
    grads = B.linear_backward(dy, B.pack8(rows), w, kept, "gelu")
    return [rows, y, r, z, *back, *grads, B.embedding_backward(dr, ids, table.shape[0])]


def step_case(rows, out, table_rows, dtype, seed=1):
    return dict(x=rand(rows, 24, dtype=dtype, seed=seed), w=rand(out, 24, dtype=dtype, seed=seed + 1, scale=0.2), b=rand(out, dtype=dtype, seed=seed + 2),
                h=rand(rows, 24, dtype=dtype, seed=seed + 3), ids=torch.randint(-1, table_rows, (rows,), device=DEV),
                table=rand(table_rows, 24, dtype=dtype, seed=seed + 4), dr=rand(rows, 24, dtype=dtype, seed=seed + 5), dy=rand(rows, out, dtype=dtype, seed=seed + 6))


CASES = [(300, 40, 9, torch.bfloat16), (70, 200, 5000, torch.bfloat16), (9000, 150, 3000, torch.float32), (16, 30, 4, torch.float32), (12000, 64, 200, torch.float16)]


@pytest.mark.parametrize("case", CASES)
def test_on_another_stream(B, case):
    c = step_case(*case)
    want = step(B, **c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:   # both at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(B, **{k: v.clone() for k, v in c.items()}))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(want, g))


@pytest.mark.parametrize("case", CASES)
def test_captured_and_replayed(B, case):
    """Two graphs, each replayed several times on new values between eager calls, against the eager results."""
    graphs = []
    for seed in (1, 50):
        c = step_case(*case, seed=seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(B, **c)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(B, **c)
        graphs.append((graph, c, out))
    for turn in range(3):
        for graph, c, out in graphs:
            for k, v in step_case(*case, seed=100 * turn + 7).items():
                c[k].copy_(v)
            graph.replay()
            want = step(B, **c)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_backward_pass_captured(B):
    r = trained(B, 32, 4, hidden=64, depth=2, dtype="bf16")
    x, views, dy = rand(500, 32, seed=1), torch.randint(0, 4, (500,), device=DEV), rand(500, 32, seed=2)
    ps = list(r.parameters())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(r(x, views), ps, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(r(x, views), ps, dy)
    for turn in range(3):
        x.copy_(rand(500, 32, seed=10 + turn))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(r(x, views), ps, dy)
        assert all(torch.equal(p, q) for p, q in zip(want, out))


# ---- sizes past 32 bits ----

@pytest.fixture
def big():
    if torch.cuda.get_device_properties(0).total_memory < 200 << 30:
        pytest.skip("needs 200 GB of device memory")
    yield
    torch.cuda.empty_cache()


def some_rows(n):
    """Rows around where 2^31 and 2^32 elements of 64 columns and 2^32 bytes end, and the last."""
    return torch.cat([torch.arange(k - 150, k + 150) for k in ((1 << 31) // 64, (1 << 32) // 64) if k + 150 < n] + [torch.arange(n - 300, n)]).to(DEV)


def test_rows_past_32_bits(B, big):
    n, T = (1 << 32) // 64 + 70001, torch.bfloat16
    base = rand(1 << 16, 64, dtype=T, seed=1)
    long = lambda shift: torch.roll(base, shift, 0).repeat(n // len(base) + 1, 1)[:n].contiguous()
    x, h, at = long(0), long(5), some_rows(n)
    one = lambda k: rand(64, dtype=T, seed=k).abs() + 0.5
    post, pre, gate = one(2), one(3), one(4)
    r, y, stats = B.residual_norm_forward(x, h, gate, post, pre)
    want = B.residual_norm_forward(x[at], h[at], gate, post, pre)
    assert torch.equal(r[at], want[0]) and torch.equal(y[at], want[1]) and torch.equal(stats[:, at], want[2])
    back = B.residual_norm_backward(x, h, r, h, gate, post, pre, stats)
    want = B.residual_norm_backward(x[at], h[at], r[at], h[at], gate, post, pre, stats[:, at].contiguous())
    assert torch.equal(back[0][at], want[0]) and torch.equal(back[1][at], want[1])
    del r, y, back
    p = B.pack8(x)
    want = B.pack8(x[at])
    assert torch.equal(p.codes[at], want.codes) and torch.equal(p.steps[at], want.steps)
    assert torch.equal(B.unpack8(p)[at], B.unpack8(want))
    w, b = rand(64, 64, dtype=T, seed=5, scale=0.1), rand(64, dtype=T, seed=6)
    y, kept = B.linear_forward(x, w, b, "gelu", h, training=True, save8=True)
    few = B.linear_forward(x[at], w, b, "gelu", h[at], training=True, save8=True)
    assert torch.equal(y[at], few[0]) and torch.equal(kept[at], few[1])
    dx, dw, db = B.linear_backward(h, p, w, kept, "gelu")
    assert torch.equal(dx[at], B.linear_backward(h[at], want, w, few[1], "gelu")[0])
    del p, y, kept, dx
    ids = torch.arange(n, device=DEV) % 300
    table = rand(300, 64, dtype=T, seed=7)
    y = B.embedding_forward(ids, table, 0.5, x)
    assert torch.equal(y[at], B.embedding_forward(ids[at], table, 0.5, x[at]))
    only = torch.full_like(ids, -1)
    only[at] = ids[at]
    got, ref = B.embedding_backward(x, only, 300), R.embedding_back(x[at], ids[at], 300, 1.0)
    R.check(got, *ref, "dtable")
    wide = B.embedding_backward(x, torch.where(only >= 0, only + 5000, only), 6000)   # by sorted positions
    R.check(wide[5000:5300], *ref, "dtable")
    assert not wide[:5000].any()


def test_features_past_32_bits(B, big):
    """Tiles: 600,000 rows of 8192 features out of 64."""
    n, T = 600000, torch.bfloat16
    x, w, b = rand(n, 64, dtype=T, seed=1), rand(8192, 64, dtype=T, seed=2, scale=0.1), rand(8192, dtype=T, seed=3)
    at = torch.cat([torch.arange(k - 300, k + 300) for k in ((1 << 31) // 8192, (1 << 32) // 8192)] + [torch.arange(n - 500, n)]).to(DEV)
    y, kept = B.linear_forward(x, w, b, "silu", training=True)
    few = B.linear_forward(x[at], w, b, "silu", training=True)
    assert torch.equal(y[at], few[0]) and torch.equal(kept[at], few[1])
    dx, dw, db = B.linear_backward(y, x, w, kept, "silu")
    ref = R.linear(x[at], w, b, "silu", None, y[at])
    R.check(dx[at], *ref["dx"], "dx")
    table = rand(700000, 8192, dtype=T, seed=4)   # a table past 2^32 elements
    ids = torch.tensor([0, 699999, 300000, 524288, 262144, 699998, 524287], device=DEV)
    assert torch.equal(B.embedding_forward(ids, table), table[ids])
    del table
    got = B.embedding_backward(y[:7].contiguous(), ids, 700000)
    assert torch.equal(got[ids], y[:7]) and int(got[:, 0].count_nonzero()) == int(y[:7, 0].count_nonzero())
