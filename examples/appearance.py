"""Trains an appearance decoder on a small scene whose images differ in exposure and tint.

    python examples/appearance.py [--steps 200]

Every step renders one image through the drop-in ops, with colours from the SH
coefficients plus the decoder's offset of each Gaussian's features, and steps the
decoder, the features and the SH coefficients on an L1 loss.  The last lines compare
with the same scene trained on its SH coefficients alone.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import tidegs_amd as tg  # noqa: E402
from tidegs_amd import scenes  # noqa: E402
from tidegs_amd.appearance import AppearanceDecoder  # noqa: E402


class Geometry:
    """The scene's projections and tile lists, which the colours do not change."""

    def __init__(self, scene):
        self.scene = scene
        means, quats, scales, self.opacities, self.sh = scenes.activations(scene.params)
        self.tiles = -(-scene.width // 16), -(-scene.height // 16)
        self.cameras = []
        for vm, K in zip(scene.viewmats, scene.Ks):
            radii, means2d, depths, conics, _ = tg.fully_fused_projection(
                means, None, quats, scales, vm[None], K[None], scene.width, scene.height)
            _, ids, flat = tg.isect_tiles(means2d, radii, depths, 16, *self.tiles)
            offsets = tg.isect_offset_encode(ids, 1, *self.tiles)
            center = torch.linalg.inv(vm)[:3, 3]
            self.cameras.append((means2d, conics, offsets, flat, (means - center)[None]))

    def render(self, camera, sh, offset=None):
        means2d, conics, tile_offsets, flat, dirs = self.cameras[camera]
        colors = tg.spherical_harmonics(3, dirs, sh[None]) + 0.5
        if offset is not None:
            colors = colors + offset[None]
        image, _ = tg.rasterize_to_pixels(means2d, conics, torch.clamp_min(colors, 0.0),
                                          self.opacities[None], self.scene.width,
                                          self.scene.height, 16, tile_offsets, flat)
        return image[0]


def targets(geometry):
    """The scene under another exposure and tint in every image."""
    out = []
    with torch.no_grad():
        for c in range(len(geometry.cameras)):
            gain = torch.tensor([1.5, 0.8, 0.5][c % 3], device="cuda")
            tint = torch.tensor([[1.0, 0.9, 0.7], [0.7, 1.0, 1.1], [1.0, 1.0, 1.0]][c % 3],
                                device="cuda")
            out.append(geometry.render(c, geometry.sh) * gain * tint)
    return out


def train(steps, decoded=True, seed=0, dtype=torch.bfloat16, say=lambda *a: None):
    """Mean L1 over the images before and after ``steps`` steps."""
    torch.manual_seed(seed)
    scene = scenes.small(seed=seed, n=4000, n_cams=6, W=160, H=96).to("cuda")
    geometry = Geometry(scene)
    images = targets(geometry)
    sh = (geometry.sh * 0.5).detach().requires_grad_()
    groups = [dict(params=[sh], lr=5e-3)]
    decoder = None
    if decoded:
        decoder = AppearanceDecoder(len(images), width=32, hidden=64, dtype=dtype).cuda()
        features = (torch.randn(scene.n, 32, device="cuda") * 0.5).requires_grad_()
        groups += [dict(params=decoder.parameters(), lr=5e-3), dict(params=[features], lr=5e-3)]
    optimizer = torch.optim.Adam(groups)

    def colors(camera, step=None):
        return decoder(features, camera, step) if decoded else None

    @torch.no_grad()
    def loss_of_all():
        if decoded:
            decoder.eval()
        losses = [(geometry.render(c, sh, colors(c)) - images[c]).abs().mean()
                  for c in range(len(images))]
        if decoded:
            decoder.train()
        return float(torch.stack(losses).mean())

    first = loss_of_all()
    for step in range(steps):
        c = step % len(images)
        loss = (geometry.render(c, sh, colors(c, step)) - images[c]).abs().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        if step % 50 == 49:
            say(f"step {step + 1}: L1 {float(loss.detach()):.4f}")
    return first, loss_of_all()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    steps = parser.parse_args().steps
    first, last = train(steps, say=print)
    print(f"with the decoder: L1 over all images {first:.4f} -> {last:.4f}")
    first, last = train(steps, decoded=False)
    print(f"SH coefficients alone: {first:.4f} -> {last:.4f}")


if __name__ == "__main__":
    main()
