"""The camera's view on its way through every mode that decodes features through a ViewRefiner."""
import dataclasses

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def trained(C, views):
    from nest_splat import residual
    r = residual.ViewRefiner(C, views, dtype="f32").to(DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    with torch.no_grad():
        for p in r.parameters():
            p.copy_(p + torch.randn(p.shape, generator=g, device=DEV) * 0.3)
    return r


@pytest.mark.parametrize("mode", ["diffuse_ngp", "diffuse_offset"])
def test_deferred_modes_decode_through_the_view_of_the_camera(mode):
    from nest_splat import renderer
    from scenes import scene
    sc = scene("shell_small")
    _, ingp = renderer.scene_to_device(sc, DEV)
    arrays = (sc.means, sc.scales, sc.rotations, sc.opacity, sc.ap_level, sc.homotrans,
              np.random.default_rng(7).normal(0, 0.5, (sc.spec.P, 16, 3)).astype(np.float32))
    means, scales, rotations, opacity, ap, homotrans, shs = (torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays)
    pc = renderer.SplatModel(means, scales, rotations, opacity, ap, homotrans=homotrans, features=shs, active_sh_degree=3)
    seen = {}
    decode = ingp.mlp_rgb.rgb_decode

    class Watched:
        def rgb_decode(self, features, ray_unit):
            seen["features"], seen["rays"] = features, ray_unit
            return decode(features, ray_unit)

    def frame(view):
        cam = dataclasses.replace(sc.cameras[0], view=view)
        return renderer.render(cam, pc, renderer.Pipe(), torch.zeros(3, device=DEV), ingp=ingp, mode=mode, with_surface=False)["ngp_rgb"]

    ingp.mlp_rgb = Watched()
    frame(None)
    plain = seen["features"]
    ingp.refiner = trained(sc.spec.C, 3)
    images = {}
    for view in (None, 0, 2):
        images[view] = frame(view)
        with torch.no_grad():
            want = ingp.refiner(plain, view)
        assert torch.equal(seen["features"], want)
        assert torch.equal(ingp.rgb_decode(plain, seen["rays"], view), decode(want, seen["rays"]))
    assert not torch.equal(images[0], images[None]) and not torch.equal(images[0], images[2])
    with pytest.raises(ValueError):
        frame(3)


def test_rgb_decode_of_no_view_and_of_a_refiner_without_views():
    from nest_splat import blocks, renderer
    from nest_splat.scene import get_spec, make_scene
    sc = make_scene(get_spec("cfg1"))
    _, ingp = renderer.scene_to_device(sc, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    features = torch.randn((70, sc.spec.C), generator=g, device=DEV)
    rays = torch.nn.functional.normalize(torch.randn((70, 3), generator=g, device=DEV), dim=-1)
    ingp.refiner = trained(sc.spec.C, 3).train()
    with torch.no_grad():
        want = ingp.mlp_rgb.rgb_decode(ingp.refiner(features), rays)
    assert torch.equal(ingp.rgb_decode(features, rays), want) and ingp.refiner.training
    ingp.refiner = blocks.GatedRefiner(sc.spec.C, dtype="f32").to(DEV)
    with pytest.raises(ValueError):
        ingp.rgb_decode(features, rays, 1)
    ingp.refiner = None
    assert torch.equal(ingp.rgb_decode(features, rays), ingp.mlp_rgb.rgb_decode(features, rays))
    with pytest.raises(ValueError):
        ingp.rgb_decode(features, rays, 1)
