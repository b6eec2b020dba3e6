"""A refiner as render() runs it: evaluation alone, in every mode that decodes features through the colour MLP."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def trained(C, **kw):
    """A refiner that changes its input."""
    from nest_splat import blocks
    r = blocks.GatedRefiner(C, depth=2, p=0.3, **kw).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    with torch.no_grad():
        for f in r.ffns:
            f.w_down.copy_(torch.randn(f.w_down.shape, generator=g, device=DEV) * 0.3)
    return r


def baseline(dtype):
    from nest_splat import renderer
    from nest_splat.scene import get_spec, make_scene
    sc = make_scene(get_spec("cfg1"))
    pc, ingp = renderer.scene_to_device(sc, DEV)
    ingp.refiner = trained(sc.spec.C, dtype=dtype)
    bg = torch.zeros(3, device=DEV)
    return ingp, lambda: renderer.render(sc.cameras[0], pc, renderer.Pipe(), bg, ingp=ingp, with_surface=False)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_render_evaluates_a_refiner_that_is_training(dtype):
    ingp, frame = baseline(dtype)
    ingp.refiner.eval()
    want = frame()["render"]
    ingp.refiner.train()
    ingp.refiner.norms[0].eval()
    state = torch.get_rng_state()
    got, again = frame()["render"], frame()["render"]
    assert torch.equal(got, want) and torch.equal(again, want)
    assert torch.equal(torch.get_rng_state(), state)
    assert ingp.refiner.training and ingp.refiner.drops[0].training and not ingp.refiner.norms[0].training


def test_render_keeps_nothing_for_a_backward_pass():
    ingp, frame = baseline("f32")
    with torch.no_grad():
        frame()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        frame()
        least = torch.cuda.max_memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = frame()
    assert torch.cuda.max_memory_allocated() <= least
    assert not out["render"].requires_grad
