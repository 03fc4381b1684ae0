"""The appearance decoder: its composition against the same in 64 bits, its dropout's
masks, and the example that trains it through the rasterizer."""
import importlib.util
from pathlib import Path

import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce
from tidegs_amd.appearance import AppearanceDecoder

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "appearance.py"
    spec = importlib.util.spec_from_file_location("appearance_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _decoder(gpu, dtype=torch.float32):
    torch.manual_seed(3)
    decoder = AppearanceDecoder(5, width=40, hidden=72, embedding=8, p=0.25, seed=11,
                                dtype=dtype).to(gpu)
    with torch.no_grad():
        decoder.head.w_down.normal_(std=0.1)
    return decoder, torch.randn(333, 40, device=gpu)


def _block64(b, x, e):
    n = torch.nn.functional
    shift = n.linear(e, b.shift.weight.double(), b.shift.bias.double())
    g, u = shift.chunk(2)
    h = n.layer_norm(x, x.shape[-1:], b.norm_weight.double(), b.norm_bias.double())
    h = n.silu(h @ b.w_gate.double().t() + g) * (h @ b.w_up.double().t() + u)
    return h @ b.w_down.double().t() + b.b_down.double()


def test_decoder_in_float32(gpu):
    """Values and every parameter's gradient against the composition in 64 bits.  Each is
    a chain of six operators whose errors are some tens of 2^-24 of their inputs' magnitudes
    (a few times the result's): 2^-24 * 6 * 40 * 4 is 6e-5."""
    announce("appearance decoder float32")
    decoder, features = _decoder(gpu)
    decoder.eval()
    leaf = features.clone().requires_grad_()
    grad = torch.randn(333, 3, device=gpu)
    out = decoder(leaf, 2)
    params = dict(decoder.named_parameters())
    got = torch.autograd.grad(out, [leaf, *params.values()], grad)
    x = leaf.double()
    e = decoder.embeddings.weight[2].double()
    want = _block64(decoder.head, x + _block64(decoder.block, x, e), e)
    exact = torch.autograd.grad(want, [leaf, *params.values()], grad.double())
    for name, a, b in (("out", out, want), *zip(["features", *params], got, exact)):
        far = float((a.double() - b.double()).norm() / b.double().norm())
        assert far < 6e-5, (name, far)


def test_decoder_draws_its_masks_from_the_step(gpu):
    announce("appearance decoder: dropout by step")
    decoder, features = _decoder(gpu, torch.bfloat16)
    with pytest.raises(ValueError, match="step"):
        decoder(features, 0)
    with torch.no_grad():
        a, b, c = decoder(features, 0, 7), decoder(features, 0, 7), decoder(features, 0, 8)
        assert a.dtype == torch.float32 and torch.equal(a, b) and not torch.equal(a, c)
        x = features.to(torch.bfloat16)
        e = decoder.embeddings.weight[0]
        h = tg.dropout(decoder.block(x, e), 0.25, 11, 7, residual=x)
        assert torch.equal(decoder.head(h, e).float(), a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_example_follows_the_exposure(gpu, dtype):
    """120 steps halve the error, which SH coefficients alone cannot: the images disagree."""
    announce(f"appearance example {dtype}")
    example = _example()
    first, last = example.train(120, dtype=dtype)
    _, alone = example.train(120, decoded=False)
    assert last < 0.5 * first and last < alone, (first, last, alone)
