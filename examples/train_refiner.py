"""Trains a GatedRefiner: the features of one scene translated to the basis that a colour head was made for.

A small synthetic scene is rendered from a view. A colour head that was trained with another grid expects its channels
mixed and bent in a fixed way, which stands here for that grid: residual blocks of layer norm, gated feed-forward and
dropout, trained with Adam on the pixels, learn it. The refiner is then set on the renderer and a frame decoded
through it.

    python examples/train_refiner.py [--steps 200] [--dtype bf16]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nest-splatting_amd"))

from nest_splat.blocks import GatedRefiner  # noqa: E402
from nest_splat.renderer import Pipe, render, scene_to_device  # noqa: E402
from nest_splat.scene import get_spec, make_scene  # noqa: E402


def train(steps: int = 200, dtype: str = "bf16", batch: int = 4096, lr: float = 3e-3, device: str = "cuda:0", log=print):
    """(refiner, loss before, loss after): mean squared errors of the whole frame's features, relative to the target's."""
    scene = make_scene(get_spec("cfg1"))
    pc, ingp = scene_to_device(scene, device)
    cam, bg = scene.cameras[0], torch.zeros(3, device=device)
    with torch.no_grad():
        features = render(cam, pc, Pipe(), bg, ingp=ingp, with_surface=False)["features"]
    C = features.shape[0]
    x = features.reshape(C, -1).t().contiguous()
    x = x / x.std()
    g = torch.Generator(device=device).manual_seed(0)
    mix = torch.linalg.qr(torch.randn(C, C, generator=g, device=device))[0]
    y = torch.tanh(x @ mix)
    refiner = GatedRefiner(C, hidden=8 * C, depth=2, p=0.02, dtype=dtype).to(device)

    def frame_loss():
        refiner.eval()
        with torch.no_grad():
            loss = (refiner(x) - y).square().mean() / y.square().mean()
        refiner.train()
        return float(loss)

    before = frame_loss()
    opt = torch.optim.Adam(refiner.parameters(), lr=lr)
    for step in range(steps):
        rows = torch.randint(0, x.shape[0], (batch,), generator=g, device=device)
        loss = (refiner(x[rows]) - y[rows]).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if step % 50 == 0:
            log(f"step {step}: loss {float(loss.detach()):.4f}")
    after = frame_loss()
    ingp.refiner = refiner.eval()
    frame = render(cam, pc, Pipe(), bg, ingp=ingp, with_surface=False)["render"]
    log(f"relative error of the features: {before:.4f} -> {after:.4f}; a frame of {tuple(frame.shape)} through the refiner")
    return refiner, before, after


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--dtype", choices=("f32", "f16", "bf16"), default="bf16")
    a = ap.parse_args()
    train(a.steps, a.dtype)
