"""Group norm with an activation, against its definition in 64 bits on the CPU.

Bounds.  u = 2^-24.  A mean or a sum over a group is taken in 32 bits over at most some tens of values
in a row and joined in trees: R = 100 u of the mean magnitude of what is summed (here |mean| + std).
So xhat is off by R kappa + R |xhat| with kappa = |mean| rstd + 1, z by |w| times that and its own
roundings, the activation by at most 1.13 times z's error and 8 u of its value (8 u |z| in gelu's and
silu's terms), and a result of 16 bits by half its step.  dz takes z's error by the slope's
slope (at most 0.8), or all of dy where relu's border lies within z's error; the sums over dz take its
errors' sums and R of their magnitudes."""
import gc

import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

U, R = 2.0 ** -24, 100 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "silu", "gelu", "relu"]
# samples, pixels, width, groups
HELD = [(1, 1, 1, 1), (1, 1, 8, 1), (2, 1, 8, 4), (3, 1, 64, 4), (1000, 1, 59, 1), (7, 16, 24, 3),
        (2, 64, 64, 8), (5, 17, 40, 5), (4, 64, 6, 6), (9, 8, 12, 3), (300, 3, 512, 32),
        (2, 4, 520, 65), (5000, 2, 16, 2), (2, 9, 512, 1), (3, 512, 8, 1), (6, 100, 31, 31),
        (4, 2, 2048, 256)]
# groups and pixels that are no whole number of vectors: overlapping ones, by teams and streamed
RAGGED = [(2000, 1, 360, 8), (50, 7, 777, 1), (3, 1, 1036, 1), (3, 1, 4124, 1), (10, 1, 2044, 1),
          (90, 3, 35, 5), (90, 3, 36, 6), (90, 3, 42, 6), (20, 30, 118, 2), (4, 200, 57, 3),
          (2, 900, 59, 1), (1, 700, 5, 5), (2, 600, 13, 1), (1, 520, 1003, 17), (1, 600, 1001, 7),
          (2, 40, 4097, 1), (2, 1100, 6, 1), (3, 2100, 2, 1), (2, 5000, 515, 5)]
STREAMED = [(4, 1, 1024, 1), (2, 1000, 64, 8), (1, 5000, 3, 1), (3, 777, 48, 6), (1, 20011, 32, 8),
            (2, 33, 1000, 4), (1, 600, 520, 1), (2, 100, 4096, 2), (40, 513, 8, 8),
            (1, 2, 65536, 2), (2, 3000, 20, 5), (1, 513, 7, 7)]


def _inputs(shape, dtype, seed=0, pitch=None, weights=None, mean=0.5):
    samples, pixels, width, _ = shape
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(samples, pixels, pitch or width, generator=g)
    x = (x * (0.5 + torch.rand(x.shape[-1], generator=g)) + mean).to(dtype).cuda()[..., :width]
    w = (1 + 0.2 * torch.randn(width, generator=g)).to(weights or dtype).cuda()
    b = (0.2 * torch.randn(width, generator=g)).to(weights or dtype).cuda()
    dy = torch.randn(samples, pixels, width, generator=g).to(dtype).cuda()
    return x, w, b, dy


def _act(name, z):
    f = torch.nn.functional
    return {None: lambda t: t, "silu": f.silu, "gelu": f.gelu, "relu": torch.relu}[name](z)


class Exact:
    """The definition in float64, and how far 32 bits may be from it."""

    def __init__(self, x, w, b, dy, groups, act, eps=1e-5):
        x, dy = x.detach().cpu().double(), dy.cpu().double()
        n, pixels, width = x.shape
        w = torch.ones(width, dtype=torch.float64) if w is None else w.detach().cpu().double()
        b = torch.zeros(width, dtype=torch.float64) if b is None else b.detach().cpu().double()

        def mean(t):  # over a sample's group, for each of its values
            t = t.view(n, pixels, groups, -1)
            return t.mean((1, 3), keepdim=True).expand(t.shape).reshape(n, pixels, width)

        mu = mean(x)
        rstd = 1 / (mean((x - mu) ** 2) + eps).sqrt()
        xh = (x - mu) * rstd
        kappa = mu.abs() * rstd + 1
        z = (xh * w + b).requires_grad_()
        y = _act(act, z)
        slope, = torch.autograd.grad(y.sum(), z)
        z, y = z.detach(), y.detach()
        dxh = R * (kappa + xh.abs())
        dz_ = w.abs() * dxh + 4 * U * ((xh * w).abs() + b.abs())
        self.y, self.far_y = y, 1.13 * dz_ + 8 * U * (y.abs() + z.abs())
        dz = dy * slope
        far = dy.abs() * (0.8 * dz_ + 8 * U * (1 + z.abs()))
        if act == "relu":
            far = torch.where(z.abs() <= dz_, dy.abs(), far)
        g, far_g = dz * w, far * w.abs()
        self.dx = rstd * (g - mean(g) - xh * mean(g * xh))
        self.far_dx = rstd * (far_g + mean(far_g) + xh.abs() * mean(far_g * xh.abs())
                              + (R + 4 * U) * (g.abs() + mean(g.abs())
                                               + xh.abs() * mean((g * xh).abs()))
                              + dxh * mean((g * xh).abs()) + xh.abs() * mean(g.abs() * dxh))
        self.dw, self.db = (dz * xh).sum((0, 1)), dz.sum((0, 1))
        self.far_dw = (far * xh.abs() + dz.abs() * dxh + R * (dz * xh).abs()).sum((0, 1))
        self.far_db = (far + R * dz.abs()).sum((0, 1))


def _near(got, want, far, what):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= far * 1.01 + half * (want.abs() + far) + tiny)
    assert not bad.any(), (what, int(bad.sum()), float((off - far)[bad].max()), off[bad][:3],
                           want[bad][:3], far[bad][:3])


def _check(x, w, b, dy, groups, act, eps=1e-5):
    exact = Exact(x, w, b, dy, groups, act, eps)
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    at = iter(leaves)
    args = [next(at) if t is not None else None for t in (x, w, b)]
    y = tg.group_norm(args[0], groups, args[1], args[2], eps, act)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(y, tg.group_norm(x, groups, w, b, eps, act))
    grads = torch.autograd.grad(y, leaves, dy)
    _near(y, exact.y, exact.far_y, "y")
    wants = [(exact.dx, exact.far_dx, "dx")]
    wants += [(exact.dw, exact.far_dw, "dw")] if w is not None else []
    wants += [(exact.db, exact.far_db, "db")] if b is not None else []
    for g, (want, far, what) in zip(grads, wants):
        _near(g, want, far, what)
    again = torch.autograd.grad(tg.group_norm(args[0], groups, args[1], args[2], eps, act),
                                leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    return grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", HELD + STREAMED + RAGGED)
def test_values_and_gradients(gpu, shape, dtype):
    act = ACTS[(sum(shape) + TYPES.index(dtype)) % 4]
    announce(f"group_norm {shape} {dtype} {act}")
    _check(*_inputs(shape, dtype), shape[3], act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40, 12, 48, 6), (2, 900, 48, 6)])
def test_activations(gpu, shape, dtype, act):
    announce(f"group_norm {shape} {dtype} {act}")
    _check(*_inputs(shape, dtype, seed=1), shape[3], act)


@pytest.mark.parametrize("shape", [(30, 12, 48, 6), (2, 900, 48, 6), (3, 50, 59, 1),
                                   (2, 1500, 59, 1)])
def test_layouts(gpu, shape):
    """Columns of wider rows, every second sample, an expanded sample, other orders of x and of dy;
    weights in 32 bits, without weights, without a bias."""
    samples, pixels, width, groups = shape
    for dtype in TYPES:
        announce(f"group_norm layouts {shape} {dtype}")
        x, w, b, dy = _inputs(shape, dtype, seed=2, pitch=width + 5)
        _check(x, w, b, dy, groups, "silu")
        wide = torch.zeros(samples, pixels, width + 3, dtype=dtype, device=gpu)
        wide[..., 1:-2] = dy
        _check(x, w, b, wide[..., 1:-2], groups, "silu")
        _check(x, w, b, dy.transpose(0, 1).contiguous().transpose(0, 1), groups, "silu")
        _check(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, dy, groups, None)
        twice = torch.stack([x, x * 2], 1).reshape(2 * samples, pixels, width)[::2]
        _check(twice, w, b, dy, groups, None)
        _check(x[:1].expand(samples, pixels, width), w, b, dy, groups, None)
        _check(x, w.float(), b.float(), dy, groups, "gelu")
        _check(x, None, b, dy, groups, "gelu")
        _check(x, w, None, dy, groups, None)
        _check(x, None, None, dy, groups, "silu")


def test_images(gpu):
    """[samples, height, width, channels], as the rasterizer leaves images, and single rows."""
    announce("group_norm of images")
    x, w, b, _ = _inputs((2, 30 * 20, 16, 4), torch.float32, seed=3)
    flat = tg.group_norm(x, 4, w, b, activation="silu")
    image = tg.group_norm(x.view(2, 30, 20, 16), 4, w, b, activation="silu")
    assert image.shape == (2, 30, 20, 16) and torch.equal(image.view(2, 600, 16), flat)
    rows = x[:, 0]
    assert torch.equal(tg.group_norm(rows, 4, w, b), tg.group_norm(x[:, :1], 4, w, b)[:, 0])
    channels_first = x.view(2, 30, 20, 16).permute(0, 3, 1, 2)  # torch's channels_last
    again = tg.group_norm(channels_first.permute(0, 2, 3, 1), 4, w, b, activation="silu")
    assert torch.equal(again, image)


def test_nothing_and_single_values(gpu):
    announce("group_norm of nothing")
    for shape in ((0, 5, 8), (2, 0, 8), (0, 8)):
        x = torch.zeros(shape, device=gpu, requires_grad=True)
        w = torch.ones(8, device=gpu, requires_grad=True)
        b = torch.ones(8, device=gpu, requires_grad=True)
        y = tg.group_norm(x, 2, w, b)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == shape and not dw.any() and not db.any()
    x = torch.full((3, 1, 4), 7.0, device=gpu)  # every group one value: its bias
    b = torch.arange(4.0, device=gpu)
    assert torch.equal(tg.group_norm(x, 4, None, b), b.expand(3, 1, 4))


def test_gradients_that_are_asked_for(gpu):
    """Each alone gives what all together give."""
    announce("group_norm: gradients one by one")
    for shape in ((40, 3, 16, 2), (2, 2000, 16, 2)):
        x, w, b, dy = _inputs(shape, torch.float32, seed=4)
        every = [t.clone().requires_grad_() for t in (x, w, b)]
        whole = torch.autograd.grad(tg.group_norm(every[0], 2, every[1], every[2],
                                                  activation="silu"), every, dy)
        for k in range(3):
            one = [t.clone().requires_grad_(k == j) for j, t in enumerate((x, w, b))]
            y = tg.group_norm(one[0], 2, one[1], one[2], activation="silu")
            assert torch.equal(torch.autograd.grad(y, one[k], dy)[0], whole[k])


def test_once_and_in_reverse_mode(gpu):
    """A second derivative and a forward tangent raise; a graph kept is used again; a tensor changed in
    place between is noticed."""
    announce("group_norm: refused derivatives")
    x, w, b, dy = _inputs((4, 50, 16, 2), torch.float32, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = tg.group_norm(leaves[0], 2, leaves[1], leaves[2], activation="silu")
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    with pytest.raises(RuntimeError, match="twice"):
        again[0].sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            tg.group_norm(dual, 2, w, b)
    y = tg.group_norm(leaves[0], 2, leaves[1], leaves[2])
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)


def test_on_another_stream(gpu):
    """Forward and backward run on the stream that is current in the forward."""
    announce("group_norm on a stream")
    x, w, b, dy = _inputs((3, 2000, 32, 4), torch.float32, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(tg.group_norm(leaves[0], 4, leaves[1], leaves[2]), leaves, dy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = leaves[0] * 1.0  # (on this stream: a launch elsewhere would not wait for it)
        got = torch.autograd.grad(tg.group_norm(late, 4, leaves[1], leaves[2]), leaves, dy)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("shape", [(4, 40, 32, 4), (4, 3000, 32, 4)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_stays_in_its_group(gpu, shape, bad):
    announce(f"group_norm with {bad} in {shape}")
    x, w, b, dy = _inputs(shape, torch.bfloat16, seed=5)
    x[2, 7, 9] = bad
    clean = x.clone()
    clean[2, 7, 9] = 0
    leaf, other = x.requires_grad_(), clean.requires_grad_()
    y, z = (tg.group_norm(t, 4, w, b, activation="silu") for t in (leaf, other))
    dx, ref = (torch.autograd.grad(t, u, dy)[0] for t, u in ((y, leaf), (z, other)))
    for a, c in ((y, z), (dx, ref)):
        assert torch.isnan(a[2, :, 8:16]).all()
        mask = torch.ones(a.shape, dtype=torch.bool, device=gpu)
        mask[2, :, 8:16] = False
        assert torch.equal(a[mask], c[mask])


@pytest.mark.parametrize("shape", [(3, 30, 16, 2), (3, 4000, 16, 2)])
def test_large_means_and_small_spreads(gpu, shape):
    """A mean of 1000 spreads costs 1000 roundings of xhat, not a million; spreads down to 1e-11."""
    announce(f"group_norm with large means {shape}")
    x, w, b, dy = _inputs(shape, torch.float32, seed=6, mean=1000.0)
    _check(x, w, b, dy, 2, None)
    x, w, b, dy = _inputs(shape, torch.float32, seed=7, mean=0.0)
    for scale, eps in ((1e-11, 2.0 ** -80), (1e-30, 2.0 ** -80), (1e15, 1e-5), (1e15, 1e20)):
        _check(x * scale, w, b, dy / 1e15, 2, None, eps)


@pytest.mark.parametrize("shape", [(6, 20, 24, 3), (2, 700, 24, 3)])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_gradient_against_differences(gpu, shape, act):
    """Along random directions; central differences of h = 1/64 are off by h^2 / 6 of third derivatives
    of order one, and by rounding: u of each y over h, in random signs."""
    announce(f"group_norm differences {shape} {act}")
    x, w, b, dy = _inputs(shape, torch.float32, seed=8)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(tg.group_norm(leaves[0], 3, leaves[1], leaves[2], activation=act),
                                leaves, dy)
    h, g = 1 / 64, torch.Generator(device="cuda").manual_seed(9)

    def value(*t):
        return float((tg.group_norm(t[0], 3, t[1], t[2], activation=act).double()
                      * dy.double()).sum())

    for k in range(3):
        v = torch.randn(leaves[k].shape, generator=g, device=gpu)
        ends = []
        for sign in (h, -h):
            t = [x, w, b]
            t[k] = t[k] + sign * v
            ends.append(value(*t))
        want = (ends[0] - ends[1]) / (2 * h)
        got = float((grads[k].double() * v.double()).sum())
        scale = float(grads[k].double().norm() * v.double().norm() / v.numel() ** 0.5)
        scale = max(scale, float(dy.double().norm()))
        assert abs(got - want) <= scale * (3 * h * h + 4 * U / h), (k, got, want)


@pytest.mark.parametrize("shape", [(50, 20, 32, 4), (2, 3000, 32, 4)])
def test_captured(gpu, shape):
    """Forward and backward in a graph, replayed with other values, between eager calls of the same
    parameters."""
    announce(f"captured group_norm {shape}")
    x, w, b, dy = _inputs(shape, torch.bfloat16, seed=10)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def both(x, w, b, dy):
        y = tg.group_norm(x, 4, w, b, activation="silu")
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*leaves, dy)
    for k in range(4):
        new = _inputs(shape, torch.bfloat16, seed=20 + k)
        with torch.no_grad():
            for t, s in zip((*leaves, dy), new):
                t.copy_(s)
        want = both(*[t.detach().clone().requires_grad_() for t in new[:3]], new[3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_captured_beside_a_living_graph(gpu):
    """Torch would end the process where a captured backward passes a gradient to a leaf of which an
    eager graph of the default stream lives: the backward raises, the forward does not, and once the
    graph is gone both are captured."""
    announce("group_norm: captured beside an eager graph")
    node = tg.decoder_ops._group_norm_node()
    x, w, b, dy = _inputs((50, 20, 32, 4), torch.bfloat16, seed=12)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def call():
        return tg.group_norm(x, 4, w, b, activation="silu")

    assert not any(map(node.gathered_by_default, leaves))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = call()
    torch.cuda.current_stream().wait_stream(side)
    assert not any(map(node.gathered_by_default, leaves))
    del kept
    kept = call()
    assert all(map(node.gathered_by_default, leaves))
    want = [kept.detach(), *torch.autograd.grad(kept, leaves, dy, retain_graph=True)]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="an eager graph of the same tensor lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(call(), leaves, dy)
    forward = torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward):
        y = call().detach()
    del kept
    gc.collect()  # (the raised error's frames)
    assert not any(map(node.gathered_by_default, leaves))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        out = [out.detach(), *torch.autograd.grad(out, leaves, dy)]
    for k in range(3):
        forward.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_past_32_bits(gpu):
    """66 samples of a million pixels and 64 channels: the last sample as it is alone (its chunks are
    others: a last bit of bfloat16 may differ)."""
    announce("group_norm of 4.3e9 values")
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.empty(66, 1_020_000, 64, dtype=torch.bfloat16, device=gpu)
    for k in (0, 64, 65):
        x[k].normal_(generator=g)
    x[1:64] = x[0]
    w = torch.ones(64, device=gpu)
    b = torch.full((64,), 0.25, device=gpu)
    leaf = x.requires_grad_()
    y = tg.group_norm(leaf, 8, w, b, activation="silu")
    dx, = torch.autograd.grad(y, leaf, y.detach())
    last = x.detach()[65:].clone().requires_grad_()
    y1 = tg.group_norm(last, 8, w, b, activation="silu")
    dx1, = torch.autograd.grad(y1, last, y1.detach())
    for a, c in ((y[65:], y1), (dx[65:], dx1)):
        off = (a.detach().float() - c.detach().float()).abs()
        assert float(off.max()) <= 2.0 ** -7 * float(c.detach().float().abs().max())
        assert float((off > 0).float().mean()) < 0.01
