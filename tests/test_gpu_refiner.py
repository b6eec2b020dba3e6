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


@pytest.mark.parametrize("mode", ["diffuse_ngp", "diffuse_offset"])
def test_deferred_modes_decode_through_the_refiner(mode):
    import numpy as np
    from nest_splat import renderer
    from scenes import scene
    sc = scene("shell_small")
    _, ingp = renderer.scene_to_device(sc, DEV)
    seen = {}

    class Watched(renderer.HashINGP):
        def __call__(self, points, with_xyz=False):
            seen["features"] = super().__call__(points, with_xyz)
            return seen["features"]

        def rgb_decode(self, features, ray_unit):
            seen["rays"] = ray_unit
            return super().rgb_decode(features, ray_unit)

    ingp.__class__ = Watched
    arrays = (sc.means, sc.scales, sc.rotations, sc.opacity, sc.ap_level, sc.homotrans,
              np.random.default_rng(7).normal(0, 0.5, (sc.spec.P, 16, 3)).astype(np.float32))
    means, scales, rotations, opacity, ap, homotrans, shs = (torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays)
    pc = renderer.SplatModel(means, scales, rotations, opacity, ap, homotrans=homotrans, features=shs, active_sh_degree=3)

    def frame():
        return renderer.render(sc.cameras[0], pc, renderer.Pipe(), torch.zeros(3, device=DEV), ingp=ingp, mode=mode, with_surface=False)

    plain = frame()["ngp_rgb"]
    ingp.refiner = trained(sc.spec.C, dtype="f32")
    got = frame()
    with torch.no_grad():
        refined = ingp.refiner.eval()(seen["features"])
    want = ingp.mlp_rgb.rgb_decode(refined, seen["rays"]).view(*got["ngp_rgb"].shape[1:], 3).permute(2, 0, 1) * (got["allmap"][1:2] > 0)
    assert torch.equal(got["ngp_rgb"], want) and not torch.equal(want, plain)
