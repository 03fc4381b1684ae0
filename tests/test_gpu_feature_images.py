"""Group norm, the gated block, the common norm and AdamW together, as they train a decoder of
rendered feature images: Gaussians' features are rasterized, normalised, decoded to colours, and
everything is stepped."""
import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce
from tidegs_amd import scenes

pytestmark = pytest.mark.gpu

WIDTH, HIDDEN, GROUPS = 16, 48, 4


def _render(scene, features, background=None):
    """Feature images [cameras, height, width, channels] of the scene's Gaussians."""
    means, quats, scales, opacities, _ = scenes.activations(scene.params)
    tiles = -(-scene.width // 16), -(-scene.height // 16)
    n = scene.viewmats.shape[0]
    radii, means2d, depths, conics, _ = tg.fully_fused_projection(
        means, None, quats, scales, scene.viewmats, scene.Ks, scene.width, scene.height)
    _, ids, flat = tg.isect_tiles(means2d, radii, depths, 16, *tiles)
    offsets = tg.isect_offset_encode(ids, n, *tiles)
    images, _ = tg.rasterize_to_pixels(means2d, conics, features.expand(n, -1, -1),
                                       opacities.expand(n, -1), scene.width, scene.height, 16,
                                       offsets, flat)
    return images


def _parameters(n, device, seed=0):
    g = torch.Generator().manual_seed(seed)

    def leaf(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(device).requires_grad_()

    return dict(features=leaf(1, n, WIDTH, scale=0.5),
                norm_w=(1 + leaf(WIDTH, scale=0.1)).detach().requires_grad_(),
                norm_b=leaf(WIDTH, scale=0.1), w_gate=leaf(HIDDEN, WIDTH, scale=0.25),
                w_up=leaf(HIDDEN, WIDTH, scale=0.25), w_down=leaf(3, HIDDEN, scale=0.15),
                b_down=leaf(3, scale=0.1))


def _decode(images, p):
    h = tg.group_norm(images, GROUPS, p["norm_w"], p["norm_b"], activation="silu")
    return tg.gated_ffn(h, p["w_gate"], p["w_up"], p["w_down"], b_down=p["b_down"])


def _decode64(images, p):
    c, h, w, k = images.shape
    x = images.view(c, h * w, GROUPS, k // GROUPS).transpose(1, 2).reshape(c, GROUPS, -1)
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    x = ((x - mean) / (var + 1e-5).sqrt()).view(c, GROUPS, h * w, -1).transpose(1, 2)
    x = torch.nn.functional.silu(x.reshape(c, h, w, k) * p["norm_w"] + p["norm_b"])
    hidden = torch.nn.functional.silu(x @ p["w_gate"].t()) * (x @ p["w_up"].t())
    return hidden @ p["w_down"].t() + p["b_down"]


def _scene(device):
    return scenes.small(seed=2, n=1500, n_cams=3, W=80, H=48).to(device)


def test_gradients_of_the_chain(gpu):
    """Of the decoder over rendered images, by what is trained, against 64 bits: a chain of five
    operators whose errors are tens of 2^-24 of their inputs' magnitudes, a few times the
    results': 5 * 40 * 4 * 2^-24 = 5e-5."""
    announce("feature images: gradients")
    scene = _scene(gpu)
    p = _parameters(scene.n, gpu)
    with torch.no_grad():
        images = _render(scene, p["features"])
    assert images.shape == (3, 48, 80, WIDTH)
    images.requires_grad_()
    decoder = {k: v for k, v in p.items() if k != "features"}
    dy = torch.randn(3, 48, 80, 3, generator=torch.Generator(device="cuda").manual_seed(1),
                     device=gpu)
    out = _decode(images, p)
    got = torch.autograd.grad(out, [images, *decoder.values()], dy)
    x = images.detach().double().requires_grad_()
    p64 = {k: v.detach().double().requires_grad_() for k, v in decoder.items()}
    want = _decode64(x, p64)
    exact = torch.autograd.grad(want, [x, *p64.values()], dy.double())
    for name, a, b in (("out", out, want), *zip(["images", *decoder], got, exact)):
        a, b = a.detach().double(), b.detach()
        far = float((a - b).norm() / b.norm())
        assert far < 5e-5, (name, far)


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_run_and_change_everything(gpu, bits):
    """Three clipped steps through the rasterizer: all parameters move, by no more than a step's
    lr (m / sqrt(v) of the first steps is at most 1 by the corrections) and decay, and a second run
    of the decoder alone gives the same bits."""
    announce(f"feature images: steps with {bits}-bit states")
    scene = _scene(gpu)
    target = torch.rand(3, 48, 80, 3, generator=torch.Generator(device="cuda").manual_seed(2),
                        device=gpu)
    p = _parameters(scene.n, gpu, seed=1)
    before = {k: v.detach().clone() for k, v in p.items()}
    opt = tg.AdamW([dict(params=[p["features"]], lr=1e-2),
                    dict(params=[v for k, v in p.items() if k != "features"])], lr=1e-3,
                   state_bits=bits, seed=7)
    for _ in range(3):
        loss = (_decode(_render(scene, p["features"]), p) - target).abs().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step(max_norm=0.5)
        assert torch.isfinite(opt.last_norm) and torch.isfinite(loss.detach())
    for k, v in p.items():
        lr = 1e-2 if k == "features" else 1e-3
        moved = (v.detach() - before[k]).abs()
        assert float(moved.max()) > 0, k
        # |m| <= sqrt(v) up to the corrections' spread over three steps; half a step of 8 bits
        assert float((moved - 3 * 1e-2 * lr * before[k].abs()).max()) <= 3 * lr * 1.5, k

    def decoded():
        q = {k: v.detach().clone().requires_grad_() for k, v in p.items()}
        one = tg.AdamW([v for k, v in q.items() if k != "features"], state_bits=bits, seed=3)
        images = torch.linspace(-1, 1, 3 * 48 * 80 * WIDTH, device=gpu).view(3, 48, 80, WIDTH)
        for _ in range(2):
            (_decode(images, q) - target).abs().mean().backward()
            one.step(max_norm=0.5)
        return q

    a, b = decoded(), decoded()
    assert all(torch.equal(a[k], b[k]) for k in a)
