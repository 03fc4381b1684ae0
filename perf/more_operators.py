"""Performance cases of what trains a network around the rasterizer: the AdamW step over
all its tensors, with its gradients clipped by their common norm and its states in 32 or
in 8 bits, and group norm with an activation over channels-last feature images.

The tensors are an appearance decoder's, the Gaussians' own tables, the features stored
with them, a wide network's; the images are a camera's 1920x1080 down to the coarse levels
of a decoder over rendered features, and rows of features that are normalised by groups.
A "forward" case is a pass without gradients (viewing), a "train" case the forward and
the backward with every gradient.
"""
from __future__ import annotations

import functools
import itertools
import math
import random

import torch

own = False  # True: the framework's operators; False: the plain forms below

LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 1e-2
BLOCK = 128  # values that share a scale where states have 8 bits
BORDER = 1.7320508  # of a block's largest value between one scale and the next
NORM_EPS = 1e-5
TABLE = (3, 1, 3, 4, 3, 45)  # values of a Gaussian: centre, opacity, scale, rotation, dc, rest


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # the last layer of a colour head: what a single call costs
        dict(name="adamw-one", kind="adamw", tensors="one", count=768, dtype="float32", bits=32,
             max_norm=0.0),
        # every step of an appearance decoder: 17 small tensors, clipped
        dict(name="adamw-decoder", kind="adamw", tensors="decoder", count=64, dtype="float32",
             bits=32, max_norm=1.0),
        # many tensors of odd sizes, packed one behind the other
        dict(name="adamw-ragged", kind="adamw", tensors="ragged", count=200, dtype="bfloat16",
             bits=32, max_norm=1.0),
        # the tables of the training configuration's 4M Gaussians
        dict(name="adamw-gaussians", kind="adamw", tensors="gaussians", count=4_000_000,
             dtype="float32", bits=32, max_norm=0.0),
        # a wide network whose states have 8 bits, clipped
        dict(name="adamw-wide-8", kind="adamw", tensors="network", count=1024, dtype="float32",
             bits=8, max_norm=1.0),
        # features of 64 values with each of 4M Gaussians, all in few bits
        dict(name="adamw-features-8", kind="adamw", tensors="rows", count=4_000_000,
             dtype="bfloat16", bits=8, max_norm=0.0),
        # the coarsest level of one image: what a single call costs
        dict(name="group-one", kind="group", samples=1, pixels=64, width=64, groups=8, pitch=64,
             dtype="bfloat16", activation="silu", train=False),
        # viewing: one camera's feature image of 1920x1080
        dict(name="group-view", kind="group", samples=1, pixels=1920 * 1080, width=32, groups=8,
             pitch=32, dtype="bfloat16", activation="silu", train=False),
        # training on four cameras' feature images at half of 1920x1080
        dict(name="group-images", kind="group", samples=4, pixels=960 * 540, width=64, groups=8,
             pitch=64, dtype="bfloat16", activation="silu", train=True),
        # 32 bits, 48 columns of wider rows, an odd image
        dict(name="group-ragged", kind="group", samples=3, pixels=241 * 137, width=48, groups=6,
             pitch=59, dtype="float32", activation="gelu", train=True),
        # the deep level of a decoder: few pixels, many channels
        dict(name="group-deep", kind="group", samples=16, pixels=30 * 34, width=512, groups=32,
             pitch=512, dtype="float16", activation="silu", train=True),
        # the feature rows of a camera's visible Gaussians, each normalised by groups
        dict(name="group-rows", kind="group", samples=1_000_000, pixels=1, width=64, groups=4,
             pitch=64, dtype="bfloat16", activation="relu", train=True),
    ]


ELEMENTS = 130_000_000  # of the largest images that are drawn


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32", "float32"])
    if rng.choice(["adamw", "group"]) == "adamw":
        tensors = rng.choice(["one", "decoder", "ragged", "gaussians", "network", "rows"])
        lo, hi = dict(one=(1, 60_000_000), decoder=(8, 512), ragged=(2, 400),
                      gaussians=(1_000, 2_000_000), network=(64, 2048),
                      rows=(1_000, 2_000_000))[tensors]
        return dict(kind="adamw", tensors=tensors, count=_log_between(rng, lo, hi), dtype=dtype,
                    bits=rng.choice([32, 8]), max_norm=rng.choice([0.0, 0.0, 1.0, 0.1]))
    groups = rng.choice([1, 2, 4, 8, 16, 32, rng.randint(1, 32)])
    rows = rng.choice([False, False, True])  # many samples of few pixels, or images
    pixels = rng.choice([1, _log_between(rng, 1, 16)]) if rows else 16
    # a group of one or two values has no gradient to speak of: 8 at least; channels of a group
    # in whole vectors half of the time (what networks have), any otherwise
    each = max(-(-8 // pixels), _log_between(rng, 1, max(8, 1024 // groups)))
    if rng.choice([False, True]):
        each = -(-each // 8) * 8
    width = groups * each
    if rows:
        samples = _log_between(rng, 1, min(1_000_000, ELEMENTS // (width * pixels)))
    else:
        samples = rng.choice([1, 1, _log_between(rng, 1, 32)])
        pixels = _log_between(rng, 16, max(17, min(1920 * 1080, ELEMENTS // (width * samples))))
    train = rng.choice([False, True])
    # relu's slope jumps where a rounding decides the sign of z: its values are drawn alone
    activation = rng.choice(["none", "silu", "silu", "gelu", "gelu" if train else "relu"])
    return dict(kind="group", samples=samples, pixels=pixels, width=width, groups=groups,
                pitch=width + rng.choice([0, 0, 0, 5]), dtype=dtype, activation=activation,
                train=train)


def _sizes(case):
    """How many values each tensor of a step has."""
    n = case["count"]
    if case["tensors"] == "one":
        return [n]
    if case["tensors"] == "rows":
        return [64 * n]
    if case["tensors"] == "gaussians":
        return [k * n for k in TABLE]
    if case["tensors"] == "network":
        return [4 * n * n, 4 * n * n, 4 * n * n, 4 * n, 4 * n, n]
    if case["tensors"] == "decoder":
        block = [n, n, 4 * n * n, 4 * n * n, 4 * n * n, n, 256 * n, 8 * n]
        return [64 * 32] + block + block[:4] + [12 * n, 3] + block[6:]
    sizes = random.Random(n)
    return [_log_between(sizes, 1, 40_000) for _ in range(n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _leaf(t, train):
    return t.detach().requires_grad_(train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    if case["kind"] == "adamw":
        return _prepare_step(case, seed, g, dtype)
    n, s, width, pitch = (case[k] for k in ("samples", "pixels", "width", "pitch"))
    # rendered features: every channel has a level and a spread of its own
    x = _randn(g, n, s, pitch) * (0.5 + torch.rand(pitch, generator=g, device="cuda"))
    x += 0.5 * _randn(g, pitch)
    train = case["train"]
    return dict(kind="group", train=train, groups=case["groups"], activation=case["activation"],
                x=_leaf(x.to(dtype)[..., :width], train),
                weight=_leaf((1 + 0.1 * _randn(g, width)).to(dtype), train),
                bias=_leaf((0.1 * _randn(g, width)).to(dtype), train),
                # the gradient that arrives from the layers above
                dy=(_randn(g, n, s, width) / 16).to(dtype) if train else None)


def _prepare_step(case, seed, g, dtype):
    """The tensors lie in flat buffers, one behind the other; with 8-bit states each of them
    begins at a block, what pads it holds zeros."""
    sizes, eight = _sizes(case), case["bits"] == 8
    spans = [-(-n // BLOCK) * BLOCK for n in sizes] if eight else sizes
    *starts, total = itertools.accumulate(spans, initial=0)
    flat = {k: torch.zeros(total, device="cuda") for k in "pgmv"}
    for start, n in zip(starts, sizes):
        # each tensor's gradients have a size of their own, its moments follow them
        size = 10 ** (-4 + 3 * float(torch.rand((), generator=g, device="cuda")))
        at = slice(start, start + n)
        flat["p"][at] = _randn(g, n) * 0.1
        flat["g"][at] = _randn(g, n) * size
        flat["m"][at] = _randn(g, n) * (0.3 * size)
        flat["v"][at] = (_randn(g, n) * 0.3 + 1).square() * size ** 2
    s = dict(kind="adamw", sizes=sizes, starts=starts, bits=case["bits"], seed=seed % (1 << 32),
             max_norm=case["max_norm"], step=500,
             p=flat["p"].to(dtype), g=flat["g"].to(dtype))
    if eight:
        s["m"], s["m_scale"] = _to_blocks(flat["m"], 8, torch.float8_e4m3fn)
        s["v"], s["v_scale"] = _to_blocks(flat["v"], 15, torch.float8_e5m2)
    else:
        s["m"], s["v"] = flat["m"], flat["v"]
    s["views"] = {k: [s[k][a:a + n] for a, n in zip(starts, sizes)] for k in "pgmv"}
    for k in ("m_scale", "v_scale"):
        s["views"][k] = [s[k][a // BLOCK:-(-(a + n) // BLOCK)]
                         for a, n in zip(starts, sizes)] if eight else None
    return s


def _exponents(most, top):
    """Of each block the power of two that brings its largest value to 2^top times 0.866 to
    1.732: below the 1.75 of the types' largest, and off what moments of few bits often are."""
    part, exponent = torch.frexp(most)
    exponent = exponent - 1 + (part >= BORDER / 2).int()
    return torch.where(most > 0, exponent - top, -120).clamp(-120, 120).int()


def _scales(flat, top):
    most = flat.view(-1, BLOCK).abs().amax(1).float()
    return ((_exponents(most, top) + 127) << 23).view(torch.float32)


def _to_blocks(flat, top, dtype):
    scale = _scales(flat, top)
    return (flat.view(-1, BLOCK) / scale[:, None]).to(dtype).view(-1), scale


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    if s["kind"] == "adamw":
        s["step"] += 1
    if not own:
        with torch.no_grad():
            return _plain_step(s) if s["kind"] == "adamw" else _plain_group(s)
    import tidegs_amd as tg

    if s["kind"] == "adamw":
        w = s["views"]
        norm = tg.grad_norm(w["g"]) if s["max_norm"] else None
        tg.adamw_step(w["p"], w["g"], w["m"], w["v"], s["step"], lr=LR, betas=BETAS, eps=EPS,
                      weight_decay=DECAY, exp_avg_scales=w["m_scale"],
                      exp_avg_sq_scales=w["v_scale"], grad_norm=norm,
                      max_norm=s["max_norm"] or None, seed=s["seed"])
        return _state(s, norm)
    activation = None if s["activation"] == "none" else s["activation"]
    y = tg.group_norm(s["x"], s["groups"], s["weight"], s["bias"], NORM_EPS, activation)
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"])]


def _state(s, norm):
    """The updated parameters and states, as they are kept."""
    out = {k: s[k] for k in ("p", "m", "v", "m_scale", "v_scale") if k in s}
    return out if norm is None else dict(out, norm=norm)


LOW = 0xFFFFFFFF


def _round(c, r, seed):
    """Round r of Philox4x32 on int64 tensors that hold 32-bit words."""
    k0 = ((seed & LOW) + r * 0x9E3779B9) & LOW
    k1 = ((seed >> 32) + r * 0xBB67AE85) & LOW
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return ((b >> 32) & LOW) ^ c[1] ^ k0, b & LOW, ((a >> 32) & LOW) ^ c[3] ^ k1, a & LOW


def _places(s):
    """(index within its tensor, its tensor's number) of each value of the flat buffers."""
    n = s["p"].numel()
    starts = torch.tensor(s["starts"], device="cuda")
    at = torch.arange(n, device="cuda")
    tensor = torch.bucketize(at, starts, right=True) - 1
    return at - starts[tensor], tensor


def _plain_draws(s):
    """16 bits for each value: half i & 1 (the low half first) of word (i & 7) >> 1 of the
    Philox4x32-10 block of counter (i >> 3, step, number of the tensor) and key `seed`."""
    i, tensor = _places(s)
    if len(s["sizes"]) == 1 and i.numel() % 8 == 0:  # one generator block for eight values
        group = i[::8] >> 3
        c = (group & LOW, group >> 32, group * 0 + s["step"], group * 0)
        words = torch.stack(functools.reduce(lambda c, r: _round(c, r, s["seed"]), range(10), c),
                            1)
        return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)
    group = i >> 3
    c = (group & LOW, group >> 32, group * 0 + s["step"], tensor)
    words = torch.stack(functools.reduce(lambda c, r: _round(c, r, s["seed"]), range(10), c), 1)
    word = words.gather(1, ((i & 7) >> 1)[:, None])[:, 0]
    return torch.where(i % 2 == 0, word & 0xFFFF, word >> 16)


def _plain_step(s):
    """g' = g min(1, max_norm / (norm + 1e-6)), m' = b1 m + (1 - b1) g',
    v' = b2 v + (1 - b2) g'^2, p' = p (1 - lr wd) - lr / (1 - b1^t) m' /
    (sqrt(v') / sqrt(1 - b2^t) + eps)."""
    (b1, b2), t = BETAS, s["step"]
    p, g = s["p"].float(), s["g"].float()
    norm = None
    if s["max_norm"]:
        norm = s["g"].double().square().sum().sqrt().float()
        g = g * torch.clamp(s["max_norm"] / (norm.double() + 1e-6), max=1.0).float()
    eight = s["bits"] == 8
    m, v = s["m"].float(), s["v"].float()
    if eight:
        m = (m.view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    p = p * (1 - LR * DECAY)
    p = p - m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + EPS) * (LR / (1 - b1 ** t))
    draws = _plain_draws(s) if eight or s["p"].dtype != torch.float32 else None
    s["p"].copy_(_plain_rounded(p, s["p"].dtype, draws))
    if eight:
        codes, scale = _to_blocks(m, 8, torch.float8_e4m3fn)
        s["m"].copy_(codes)
        s["m_scale"].copy_(scale)
        s["v_scale"].copy_(_scales(v, 15))
        s["v"].copy_(_plain_second(v, s["v_scale"], draws))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _state(s, norm)


def _plain_rounded(p, dtype, draws):
    """p in 16 bits: up with the probability of what lies below the last bit."""
    if dtype == torch.float32:
        return p
    if dtype == torch.bfloat16:
        return ((p.view(torch.int32) + draws.int()) & -65536).view(torch.float32).to(dtype)
    # below 2^-14 half precision's steps no longer shrink: 2^-14 more has their spacing
    lift = torch.where(p.abs() < 2.0 ** -14, 2.0 ** -14, 0.0)
    a = ((p.abs() + lift).view(torch.int32) + (draws >> 3).int()) & -8192
    return torch.copysign(a.view(torch.float32) - lift, p).to(dtype)


def _plain_second(v, scale, draws):
    """v in units of its block's scale in e5m2, up with the probability of what lies below the
    last bit; a positive one never to 0."""
    x = (v.view(-1, BLOCK) / scale[:, None]).view(-1)
    lift = torch.where(x < 2.0 ** -14, 2.0 ** -14, 0.0)
    a = ((x + lift).view(torch.int32) + (draws * 32 + 16).int()) & -(1 << 21)
    a = a.view(torch.float32) - lift
    return torch.where(x > 0, a.clamp(min=2.0 ** -16), 0.0).to(torch.float8_e5m2)


def _activation(name, z):
    """act(z) and act'(z)."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if name == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _plain_group(s):
    """y = act(z), z = xhat w + b with xhat = (x - mean) rstd over a sample's group; with
    dz = dy act'(z) and g = dz w: dx = rstd (g - mean(g) - xhat mean(g xhat))."""
    n, pixels, width = s["x"].shape
    split = (n, pixels, s["groups"], width // s["groups"])
    x = s["x"].float().reshape(split)
    w, b = (s[k].float().view(split[2:]) for k in ("weight", "bias"))
    over = (1, 3)
    d = x - x.mean(over, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(over, keepdim=True) + NORM_EPS)
    xhat = d * rstd
    y, slope = _activation(s["activation"], xhat * w + b)
    dtype = s["x"].dtype
    y = y.to(dtype).view(n, pixels, width)
    if not s["train"]:
        return [y]
    dz = s["dy"].float().view(split) * slope
    g = dz * w
    dx = rstd * (g - g.mean(over, keepdim=True) - xhat * (g * xhat).mean(over, keepdim=True))
    return [y, dx.to(dtype).view(n, pixels, width),
            (dz * xhat).sum((0, 1)).view(-1).to(dtype), dz.sum((0, 1)).view(-1).to(dtype)]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_step(s) if s["kind"] == "adamw" else _exact_group(s)


def _exact_group(s):
    x, w, b = (s[k].detach().double().requires_grad_(s["train"]) for k in ("x", "weight", "bias"))
    act = dict(none=lambda z: z, silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu,
               relu=torch.relu)[s["activation"]]
    n, pixels, width = x.shape
    rows = x.view(n, pixels, s["groups"], -1).transpose(1, 2).reshape(n, s["groups"], -1)
    var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
    rows = ((rows - mean) / (var + NORM_EPS).sqrt()).view(n, s["groups"], pixels, -1)
    y = act(rows.transpose(1, 2).reshape(n, pixels, width) * w + b)
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [x, w, b], s["dy"].double())]


def _mul_words(a, k):
    """(high, low) 32-bit words of a * k from 16-bit parts."""
    a0, a1, k0, k1 = a & 0xFFFF, a >> 16, k & 0xFFFF, k >> 16
    mid = a1 * k0 + ((a0 * k0) >> 16)
    mid2 = a0 * k1 + (mid & 0xFFFF)
    return a1 * k1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((a0 * k0) & 0xFFFF)


def _exact_draws(n, tensor, step, seed):
    i = torch.arange(n, device="cuda")
    c = [(i >> 3) & LOW, i >> 35, torch.full_like(i, step), torch.full_like(i, tensor)]
    key = [seed % (1 << 32), seed >> 32]
    for _ in range(10):
        h0, l0 = _mul_words(c[0], 0xD2511F53)
        h1, l1 = _mul_words(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    part = i & 7
    word = torch.where(part < 4, torch.where(part < 2, c[0], c[1]),
                       torch.where(part < 6, c[2], c[3]))
    return torch.where(part % 2 == 0, word % 65536, word // 65536)


def _exact_blocks(x, top):
    """x by blocks and each block's scale."""
    rows = torch.nn.functional.pad(x, (0, -len(x) % BLOCK)).view(-1, BLOCK)
    most = rows.abs().amax(1, keepdim=True)
    exponent = torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / BORDER)) - top
    return rows, torch.exp2(torch.where(most > 0, exponent, -120.0).clamp(-120, 120))


def _grid(x, lowest, bits):
    """The spacing at x of floats with that many stored bits and normal numbers from 2^lowest."""
    size = torch.floor(torch.log2(torch.where(x == 0, 1.0, x.abs())))
    size = torch.where(x == 0, float(lowest), size)
    return torch.exp2(size.clamp(min=lowest) - bits)


def _exact_step(s):
    """By the formula, tensor by tensor; the parameters before their rounding."""
    (b1, b2), t = BETAS, s["step"] + 1
    clip, norm = 1.0, None
    if s["max_norm"]:
        norm = torch.stack([g.double().norm() for g in s["views"]["g"]]).norm()
        clip = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    keys = ("p", "m", "v") + (("m_scale", "v_scale") if s["bits"] == 8 else ())
    out = {k: torch.zeros(s[k].shape, dtype=torch.float64, device="cuda") for k in keys}
    for k, (start, n) in enumerate(zip(s["starts"], s["sizes"])):
        p, g, m, v = (s["views"][name][k].double() for name in "pgmv")
        at, blocks = slice(start, start + n), slice(start // BLOCK, -(-(start + n) // BLOCK))
        if s["bits"] == 8:
            m = m * s["m_scale"][blocks].double().repeat_interleave(BLOCK)[:n]
            v = v * s["v_scale"][blocks].double().repeat_interleave(BLOCK)[:n]
        g = g * clip
        m = m + (1 - b1) * (g - m)
        v = v + (1 - b2) * (g * g - v)
        out["p"][at] = p - LR * DECAY * p \
            - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        if s["bits"] == 8:
            rows, scale = _exact_blocks(m, 8)
            x = (rows / scale).view(-1)[:n]
            step = _grid(x, -6, 3)
            m, out["m_scale"][blocks] = torch.round(x / step) * step, scale[:, 0]
            rows, scale = _exact_blocks(v, 15)
            x = (rows / scale).view(-1)[:n]
            step = _grid(x, -14, 2)
            up = (_exact_draws(n, k, t, s["seed"]) + 0.5) / 65536
            v = torch.where(x > 0, (torch.floor(x / step + up) * step).clamp(min=2.0 ** -16), 0.0)
            out["v_scale"][blocks] = scale[:, 0]
        out["m"][at], out["v"][at] = m, v
    return out if norm is None else dict(out, norm=norm)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "adamw":
        # the gradient in, the parameter and both states in and out, scales with 8-bit states
        n, state = sum(_sizes(case)), 4 if case["bits"] == 32 else 1 + 4 / BLOCK
        return dict(bytes=n * (3 * size + 4 * state), flops=(18 if case["max_norm"] else 16) * n)
    n, train = case["samples"] * case["pixels"] * case["width"], case["train"]
    # x in, y out; backward: x and dy in, dx out; the weights and their gradients
    return dict(bytes=size * (5 if train else 2) * (n + case["width"]),
                flops=(40 if train else 12) * n)
