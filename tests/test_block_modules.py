"""The decoder block's modules as programs use them: recomputed forwards, copies, seeds. On the CPU a mask of torch's stands in
for the library's, as a function of the seed and the offset alone."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint


@pytest.fixture
def B(monkeypatch):
    from nest_splat import blocks

    def masked(x, p, seed, offset=0, residual=None):
        g = torch.Generator().manual_seed((seed * 1000003 + offset) % (1 << 63))
        y = torch.where(torch.rand(x.shape, generator=g) >= p, x / (1 - p), torch.zeros(()))
        return y if residual is None else residual + y

    monkeypatch.setattr(blocks, "dropout_forward", masked)
    return blocks


def masks(drop, n, size=4096):
    return [drop(torch.ones(size)) != 0 for _ in range(n)]


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_recomputed_forward_draws_the_same_mask(B, reentrant):
    drops = [B.Dropout(0.4), B.Dropout(0.4)]

    def block(x):
        return drops[1](torch.sin(drops[0](x)), residual=x)

    torch.manual_seed(5)
    x = torch.randn(300, requires_grad=True)
    state = torch.get_rng_state()
    want = torch.autograd.grad(block(x).square().sum(), x)[0]
    torch.set_rng_state(state)
    checkpoint(block, x, use_reentrant=reentrant).square().sum().backward()
    assert torch.equal(x.grad, want)


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_counted_mask_refuses_to_be_recomputed(B, reentrant):
    drop = B.Dropout(0.4, seed=3)
    x = torch.randn(300, requires_grad=True)
    y = checkpoint(lambda t: torch.sin(drop(t)), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="recomputed"):
        y.sum().backward()
    assert drop.offset == 1
    torch.autograd.grad(drop(x).sum(), x)  # a plain step goes on


def test_modules_without_a_seed_follow_torch(B):
    torch.manual_seed(1)
    a, b = B.Dropout(0.5), B.Dropout(0.5)
    first = masks(a, 2) + masks(b, 2)
    assert all(not torch.equal(p, q) for i, p in enumerate(first) for q in first[:i])
    torch.manual_seed(1)
    assert all(torch.equal(p, q) for p, q in zip(first, masks(a, 2) + masks(b, 2)))
    torch.manual_seed(2)
    assert not torch.equal(first[0], masks(a, 1)[0])


def test_a_seed_makes_a_sequence_of_its_own_that_the_state_dict_keeps(B):
    a, b = B.Dropout(0.5, seed=9), B.Dropout(0.5)
    torch.manual_seed(1)
    want = masks(a, 3)
    torch.manual_seed(2)
    assert all(torch.equal(p, q) for p, q in zip(want, masks(B.Dropout(0.5, seed=9), 3)))
    b.load_state_dict(a.state_dict())
    assert torch.equal(masks(b, 1)[0], masks(copy.deepcopy(a), 1)[0])
    plain = B.Dropout(0.5)
    b.load_state_dict(plain.state_dict())
    assert b.seed is None


def test_replicas_of_a_counted_module_are_refused(B):
    """A replica counts on a copy that is thrown away, so every step would draw the first masks again."""
    x = torch.ones(8)
    with pytest.raises(RuntimeError, match="replica"):
        B.Dropout(0.5, seed=1)._replicate_for_data_parallel()(x)
    B.Dropout(0.5)._replicate_for_data_parallel()(x)
    B.Dropout(0.5, seed=1).eval()._replicate_for_data_parallel()(x)


def test_blocks_of_a_refiner_have_masks_of_their_own(B):
    torch.manual_seed(0)
    drops = [d for _ in range(2) for d in B.GatedRefiner(16, depth=2, p=0.5).drops]
    seen = [masks(d, 1)[0] for d in drops]
    assert all(not torch.equal(p, q) for i, p in enumerate(seen) for q in seen[:i])


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed_blocks_have_the_gradients_of_kept_ones(reentrant):
    from nest_splat import blocks
    dev = torch.device("cuda:0")
    refiner = blocks.GatedRefiner(32, depth=2, p=0.3, dtype="f32").to(dev)
    with torch.no_grad():
        for f in refiner.ffns:
            f.w_down.normal_(0, 0.3)
    x = torch.randn(500, 32, device=dev, requires_grad=True)

    def grads(run):
        torch.manual_seed(4)
        return torch.autograd.grad(run().square().sum(), [x, *refiner.parameters()])

    want = grads(lambda: refiner(x))
    if reentrant:  # grad() does not go through it
        torch.manual_seed(4)
        checkpoint(refiner, x, use_reentrant=True).square().sum().backward()
        got = [x.grad, *(p.grad for p in refiner.parameters())]
    else:
        got = grads(lambda: checkpoint(refiner, x, use_reentrant=False))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


class _Recorder:
    """Stands in for the library: sizes and calls of the gated feed-forward block, on the CPU."""

    def __init__(self, blocks, monkeypatch):
        self.kept = []
        monkeypatch.setattr(blocks, "gated_ffn_forward", self.forward)

    def forward(self, x, w_gate, w_up, w_down, activation="silu", training=False):
        self.kept.append(training)
        return x @ w_down.t() if x.shape[-1] == w_down.shape[1] else x.new_zeros(x.shape[0], w_down.shape[0]), None


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_forward_without_gradients_keeps_nothing_for_them(monkeypatch, mode):
    """Under no_grad a parameter still asks for its gradient, but there will be none."""
    from nest_splat import blocks
    seen = _Recorder(blocks, monkeypatch)
    ffn = blocks.GatedFFN(8, 16, dtype="f32")
    x = torch.zeros(4, 8)
    with mode():
        ffn(x)
    blocks.gated_ffn(x, *(w.detach() for w in ffn.parameters()))
    assert seen.kept == [False, False]
    assert ffn(x).requires_grad
    assert seen.kept[2]
