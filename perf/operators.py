"""Performance cases of the decoder operators: layer norm, dropout and the gated
feed-forward block, the parts of a small network that turns the features stored
with each Gaussian into its colour.

The ordinary rows are Gaussians: a camera's visible ones, a working set of 4096-row
blocks, the 4M of the training configuration; ordinary widths are those of the
resident table (59 columns at a pitch of 64), of 16 SH coefficients of three
channels (48) and of RGB (3), beside the powers of two of generic networks.  A
"forward" case is a pass without gradients (viewing), a "train" case the forward
and the backward with every gradient.
"""
from __future__ import annotations

import functools
import math

import torch

own = False  # True: the framework's operators; False: the plain forms below

TABLE_COLUMNS, TABLE_PITCH = 59, 64
ELEMENTS = 256_000_000  # of the largest element-wise cases: 4M rows of 64


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # the norm of one row: what a single call costs
        dict(name="norm-one", kind="norm", rows=1, width=64, pitch=64, dtype="bfloat16",
             train=False),
        # rows of a resident table as they lie there: 59 columns at a pitch of 64
        dict(name="norm-table", kind="norm", rows=300_001, width=59, pitch=64, dtype="float32",
             train=True),
        # the features of all 4M Gaussians of the training configuration
        dict(name="norm-features", kind="norm", rows=4_000_000, width=64, pitch=64,
             dtype="bfloat16", train=True),
        # a wide network over the tokens of images
        dict(name="norm-wide", kind="norm", rows=8_191, width=1024, pitch=1024, dtype="float16",
             train=True),
        # dropout of one camera's image embedding
        dict(name="drop-one", kind="drop", rows=1, width=64, dtype="float32", p=0.1,
             residual=False, train=False),
        # a working set's rows of 59 columns, nothing aligned
        dict(name="drop-ragged", kind="drop", rows=300_001, width=59, dtype="float32", p=0.2,
             residual=False, train=True),
        # a residual branch over the features of all 4M Gaussians
        dict(name="drop-features", kind="drop", rows=4_000_000, width=64, dtype="bfloat16", p=0.1,
             residual=True, train=True),
        # one row through a wide network: the weights' bytes are the work
        dict(name="ffn-one", kind="ffn", rows=1, width=1024, hidden=4096, out=1024, pitch=1024,
             dtype="bfloat16", activation="silu", bias=False, train=False),
        # viewing: SH coefficients of a camera's visible Gaussians
        dict(name="ffn-colours", kind="ffn", rows=1_000_000, width=64, hidden=256, out=48,
             pitch=64, dtype="bfloat16", activation="silu", bias=True, train=False),
        # training in 32 bits from the table's own rows to RGB
        dict(name="ffn-table", kind="ffn", rows=300_001, width=59, hidden=128, out=3, pitch=64,
             dtype="float32", activation="gelu", bias=True, train=True),
        # training a residual block over a camera's visible Gaussians
        dict(name="ffn-features", kind="ffn", rows=1_000_000, width=64, hidden=256, out=64,
             pitch=64, dtype="bfloat16", activation="silu", bias=True, train=True),
        # training a wide network over the tokens of images
        dict(name="ffn-wide", kind="ffn", rows=8_192, width=1024, hidden=4096, out=1024,
             pitch=1024, dtype="bfloat16", activation="silu", bias=False, train=True),
    ]


def _log_between(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(["norm", "drop", "ffn", "ffn"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.choice([False, True])
    if kind == "ffn":
        # widths in steps of 8 half of the time (what networks have), any otherwise
        width, hidden = _log_between(rng, 16, 1024), _log_between(rng, 32, 4096)
        if rng.choice([False, True]):
            width, hidden = -(-width // 8) * 8, -(-hidden // 8) * 8
        hidden += 8 * (hidden == 3072)
        out = rng.choice([3, 48, width, _log_between(rng, 3, 1024)])
        products = 2 * (2 * width * hidden + hidden * out) * (3 if train else 1)
        # no more work than the largest listed case, no more hidden values either
        most = min(1_000_000, ELEMENTS // hidden, int(6e11 / products))
        if dtype == "float32":
            most = max(1, most // 4)
        return dict(kind=kind, rows=_log_between(rng, 1, most), width=width, hidden=hidden,
                    out=out, pitch=width + rng.choice([0, 0, 5]), dtype=dtype,
                    activation=rng.choice(["silu", "gelu", "relu"]),
                    bias=rng.choice([False, True]), train=train)
    width = rng.choice([TABLE_COLUMNS, 64, _log_between(rng, 3, 4096), _log_between(rng, 3, 4096)])
    most = ELEMENTS // (2 if dtype == "float32" else 1) // width
    case = dict(kind=kind, rows=_log_between(rng, 1, min(4_000_000, most)), width=width,
                dtype=dtype, train=train)
    if kind == "norm":
        case["pitch"] = TABLE_PITCH if width == TABLE_COLUMNS else width + rng.choice([0, 0, 3])
    else:
        case["p"] = rng.choice([0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 4)])
        case["residual"] = rng.choice([False, True])
    return case


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
    n, width = case["rows"], case["width"]
    pitch = case.get("pitch", width)
    # learned features: every column has a level and a spread of its own
    rows = _randn(g, n, pitch) * (0.5 + torch.rand(pitch, generator=g, device="cuda"))
    rows += 0.3 * _randn(g, pitch)
    s = dict(kind=case["kind"], train=case["train"],
             x=_leaf(rows.to(dtype)[:, :width], case["train"]))
    del rows
    out = width
    if case["kind"] == "norm":
        s["weight"] = _leaf((1 + 0.1 * _randn(g, width)).to(dtype), case["train"])
        s["bias"] = _leaf((0.1 * _randn(g, width)).to(dtype), case["train"])
    elif case["kind"] == "drop":
        s.update(p=case["p"], seed=seed * 0x9E3779B97F4A7C15 % (1 << 63), offset=seed % 1000,
                 residual=None)
        if case["residual"]:
            s["residual"] = _leaf(_randn(g, n, width).to(dtype), case["train"])
    else:
        out, hidden = case["out"], case["hidden"]
        s["activation"] = case["activation"]
        weights = dict(w_gate=(hidden, width), w_up=(hidden, width), w_down=(out, hidden))
        for name, (a, b) in weights.items():
            s[name] = _leaf((_randn(g, a, b) / math.sqrt(b)).to(dtype), case["train"])
            s["b" + name[1:]] = _leaf((0.1 * _randn(g, a)).to(dtype), case["train"]) \
                if case["bias"] else None
    # the gradient that arrives from the layers above
    s["dy"] = (_randn(g, n, out) / 16).to(dtype) if case["train"] else None
    return s


def _inputs(s):
    """What a case differentiates by, in the order of the outputs after y."""
    names = {"norm": ("x", "weight", "bias"), "drop": ("x", "residual"),
             "ffn": ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")}[s["kind"]]
    return [s[name] for name in names if s[name] is not None]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    if not own:
        with torch.no_grad():
            return PLAIN[s["kind"]](s)
    import tidegs_amd as tg

    if s["kind"] == "norm":
        y = tg.layer_norm(s["x"], s["weight"], s["bias"])
    elif s["kind"] == "drop":
        y = tg.dropout(s["x"], s["p"], s["seed"], offset=s["offset"], residual=s["residual"])
    else:
        y = tg.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"],
                         s["b_down"], activation=s["activation"])
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, _inputs(s), s["dy"])]


EPS = 1e-5


def _plain_norm(s):
    """y = xhat w + b with xhat = (x - mean) rstd; dx = rstd (g - mean(g) - xhat mean(g xhat))
    with g = dy w."""
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    xhat = d * rstd
    y = xhat * w + b
    dtype = s["x"].dtype
    if not s["train"]:
        return [y.to(dtype)]
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return [t.to(dtype) for t in (y, dx, (dy * xhat).sum(0), dy.sum(0))]


LOW = 0xFFFFFFFF


def _round(c, r, seed):
    """Round r of Philox4x32 on int64 tensors that hold 32-bit words."""
    k0 = ((seed & LOW) + r * 0x9E3779B9) & LOW
    k1 = ((seed >> 32) + r * 0xBB67AE85) & LOW
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return ((b >> 32) & LOW) ^ c[1] ^ k0, b & LOW, ((a >> 32) & LOW) ^ c[3] ^ k1, a & LOW


def _plain_keep(n, p, seed, offset, device):
    """Which of n values dropout keeps: the 16-bit draw of value i is half i & 1 (the low
    half first) of word (i & 7) >> 1 of the Philox4x32-10 block of counter (i >> 3, offset) and
    key `seed`; the value stays where its draw is not below p in 65536ths."""
    group = torch.arange(-(-n // 8), device=device)
    zero = torch.zeros_like(group)
    c = (group & LOW, group >> 32, zero + (offset & LOW), zero + (offset >> 32))
    c = functools.reduce(lambda c, r: _round(c, r, seed), range(10), c)
    words = torch.stack(c, 1)
    draws = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    return draws >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _plain_drop(s):
    x = s["x"].float()
    keep = _plain_keep(x.numel(), s["p"], s["seed"], s["offset"], x.device).view(x.shape)
    scale = 65536 / (65536 - _threshold(s["p"]))
    y = torch.where(keep, x * scale, 0.0)
    dtype, residual = s["x"].dtype, s["residual"]
    if residual is not None:
        y = y + residual.float()
    if not s["train"]:
        return [y.to(dtype)]
    dx = torch.where(keep, s["dy"].float() * scale, 0.0)
    return [y.to(dtype), dx.to(dtype)] + ([s["dy"].clone()] if residual is not None else [])


def _activation(name, g):
    """act(g) and act'(g)."""
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if name == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _plus(t, b):
    return t if b is None else t + b.float()


def _plain_ffn(s):
    """y = h Wd^T + bd with h = act(g) u, g = x Wg^T + bg, u = x Wu^T + bu."""
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = _plus(x @ wg.t(), s["b_gate"]), _plus(x @ wu.t(), s["b_up"])
    a, da = _activation(s["activation"], g)
    h = a * u
    y = _plus(h @ wd.t(), s["b_down"])
    dtype = s["x"].dtype
    if not s["train"]:
        return [y.to(dtype)]
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    grads = [dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h]
    if s["b_gate"] is not None:
        grads += [dg.sum(0), du.sum(0), dy.sum(0)]
    return [t.to(dtype) for t in [y, *grads]]


PLAIN = dict(norm=_plain_norm, drop=_plain_drop, ffn=_plain_ffn)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _mul_words(a, k):
    """(high, low) 32-bit words of a * k from 16-bit parts."""
    a0, a1, k0, k1 = a & 0xFFFF, a >> 16, k & 0xFFFF, k >> 16
    mid = a1 * k0 + ((a0 * k0) >> 16)
    mid2 = a0 * k1 + (mid & 0xFFFF)
    return a1 * k1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((a0 * k0) & 0xFFFF)


def _draws64(n, seed, offset):
    i = torch.arange(n, device="cuda")
    c = [(i >> 3) & LOW, i >> 35, torch.full_like(i, offset & LOW),
         torch.full_like(i, offset >> 32)]
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


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double().requires_grad_(s["train"])
         if isinstance(v, torch.Tensor) and k != "dy" else v for k, v in s.items()}
    x = d["x"]
    if s["kind"] == "norm":
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / (var + EPS).sqrt() * d["weight"] + d["bias"]
    elif s["kind"] == "drop":
        t = round(s["p"] * 65536)
        draws = _draws64(x.numel(), s["seed"], s["offset"]).view(x.shape)
        y = x.masked_fill(draws < t, 0) / (1 - t / 65536)
        y = y if d["residual"] is None else y + d["residual"]
    else:
        act = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu,
                   relu=torch.relu)[s["activation"]]
        linear = torch.nn.functional.linear
        h = act(linear(x, d["w_gate"], d["b_gate"])) * linear(x, d["w_up"], d["b_up"])
        y = linear(h, d["w_down"], d["b_down"])
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, _inputs(d), s["dy"].double())]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    n, width, train = case["rows"], case["width"], case["train"]
    if case["kind"] == "norm":
        # x in, y out; backward: x and dy in, dx out; the weights and their gradients
        return dict(bytes=size * ((5 if train else 2) * n * width + (5 if train else 2) * width),
                    flops=(20 if train else 8) * n * width)
    if case["kind"] == "drop":
        # x in, y out; backward: dy in, dx out; the residual in, its gradient out
        moved = 4 if train else 2
        moved += (2 if train else 1) if case["residual"] else 0
        return dict(bytes=size * moved * n * width, flops=2 * n * width)
    hidden, out = case["hidden"], case["out"]
    weights = 2 * hidden * width + hidden * out + (2 * hidden + out if case["bias"] else 0)
    # forward: x and the weights in, y out; backward: x, dy and the weights in, their gradients out
    moved = n * (width + out) + weights
    if train:
        moved += n * (2 * width + out) + 2 * weights
    return dict(bytes=size * moved,
                flops=2 * n * (2 * width * hidden + hidden * out) * (3 if train else 1))
