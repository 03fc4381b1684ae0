"""The decoder operators against their definitions in 64 bits.

Tolerances are bounds, element by element, from the operators' own rounding: ``u`` is
the unit roundoff of the tensors' type, a sum of n products in 32 bits is off by
at most (n + 8) 2^-24 times the sum of their magnitudes, and each error is carried
through the formulas to the outputs in 64 bits beside the values.
"""
import math

import numpy as np
import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
# what rounding loses, or a flush to zero takes, below a type's normal range
FLOOR = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gamma(n):
    return (n + 8) * U32


def _within(got, want, bound, what):
    """Every element of ``got`` within ``bound`` of ``want``."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    far = (got.double() - want).abs() - bound
    assert bool((far <= 0).all()), \
        f"{what}: {int((~(far <= 0)).sum())} of {far.numel()} values out, by {float(far.max()):.3g}"


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------


def _norm64(x, w, b, eps, dy=None):
    """Values and error bounds of y (and dx, dw, db), from 64-bit copies of the inputs."""
    u = UNIT[x.dtype]
    n = x.shape[-1]
    tiny = FLOOR[x.dtype]
    uw, tiny_w = (u, tiny) if w is None else (UNIT[w.dtype], FLOOR[w.dtype])
    x = x.double()
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    xhat = d * rstd
    # the mean is off by gamma times the mean magnitude, each difference by that and a rounding;
    # the second pass's sum of squares by twice the differences' error
    e_mean = _gamma(n) * x.abs().mean(-1, keepdim=True)
    e_d = e_mean + U32 * (x.abs() + mean.abs())
    e_rstd = rstd * (_gamma(n) + (d.abs() * e_d).mean(-1, keepdim=True) * rstd ** 2)
    e_xhat = e_d * rstd + d.abs() * e_rstd + 2 * U32 * xhat.abs()
    y = xhat * w + b
    e_y = e_xhat * w.abs() + 2 * U32 * (xhat * w).abs() + U32 * b.abs() + u * y.abs() + tiny
    if dy is None:
        return [(y, e_y)]
    dy = dy.double()
    g = dy * w
    mg, mgx = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
    e_mg = (_gamma(n) + U32) * g.abs().mean(-1, keepdim=True)
    e_mgx = ((_gamma(n) + U32) * (g * xhat).abs() + g.abs() * e_xhat).mean(-1, keepdim=True)
    inner = g - mg - xhat * mgx
    size = g.abs() + mg.abs() + (xhat * mgx).abs()
    dx = rstd * inner
    e_dx = rstd * (e_mg + e_xhat * mgx.abs() + xhat.abs() * e_mgx + 4 * U32 * size) \
        + inner.abs() * e_rstd + u * dx.abs() + tiny
    rows = x.shape[0]
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    e_dw = _gamma(rows) * (dy * xhat).abs().sum(0) + (dy.abs() * e_xhat).sum(0) + uw * dw.abs()
    e_db = _gamma(rows) * dy.abs().sum(0) + uw * db.abs()
    return [(y, e_y), (dx, e_dx), (dw, e_dw + tiny_w), (db, e_db + tiny_w)]


NORM_SHAPES = [(1, 1), (1, 64), (3, 5), (17, 16), (5, 17), (300, 59), (257, 64), (33, 72),
               (4097, 64), (1000, 65), (64, 128), (9, 264), (130, 512), (31, 1000), (12, 1024),
               (7, 2047), (5, 2304), (6, 4096), (3, 4097), (2, 9001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_layer_norm(gpu, rows, width, dtype):
    announce(f"layer norm {rows}x{width} {dtype}")
    g = _gen(rows * 7919 + width)
    x = (_rand(g, rows, width) * (0.5 + torch.rand(width, generator=g, device=gpu))
         + 0.5).to(dtype).requires_grad_()
    w, b = _rand(g, width, dtype=dtype).requires_grad_(), _rand(g, width, dtype=dtype).requires_grad_()
    dy = _rand(g, rows, width, dtype=dtype)
    y = tg.layer_norm(x, w, b, 1e-5)
    got = [y, *torch.autograd.grad(y, (x, w, b), dy)]
    want = _norm64(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for t, (v, e), name in zip(got, want, ("y", "dx", "dw", "db")):
        assert t.dtype == dtype
        _within(t, v, e, f"{name} of {rows}x{width}")
    with torch.no_grad():
        assert torch.equal(tg.layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pitch,first,width", [(64, 0, 59), (64, 4, 40), (67, 0, 64), (128, 64, 64),
                                               (1100, 3, 1024), (5000, 1, 4500)])
def test_layer_norm_columns_of_a_table(gpu, pitch, first, width, dtype):
    announce(f"layer norm of columns {first}:{first + width} at pitch {pitch} {dtype}")
    g = _gen(pitch + width)
    table, grads = (_rand(g, 45, pitch, dtype=dtype) for _ in range(2))
    x = table[:, first:first + width].detach().requires_grad_()
    dy = grads[:, first:first + width]
    w = _rand(g, width).requires_grad_()  # float32 weights of x of any type
    y = tg.layer_norm(x, w, None, 1e-3)
    got = [y, *torch.autograd.grad(y, (x, w), dy)]
    for t, (v, e), name in zip(got, _norm64(x.detach(), w.detach(), None, 1e-3, dy),
                               ("y", "dx", "dw")):
        _within(t, v, e, name)
    assert got[2].dtype == torch.float32


def test_layer_norm_shapes_and_absent_parts(gpu):
    announce("layer norm: batch shapes, no weights, no rows")
    g = _gen(5)
    x = _rand(g, 3, 4, 5, 24)
    y = tg.layer_norm(x)
    _within(y.view(-1, 24), *_norm64(x.view(-1, 24), None, None, 1e-5)[0], "4d")
    b = _rand(g, 24).requires_grad_()
    y = tg.layer_norm(x.transpose(0, 2), bias=b)
    assert y.shape == (5, 4, 3, 24)
    _within(y.reshape(-1, 24), *_norm64(x.transpose(0, 2).reshape(-1, 24), None, b.detach(), 1e-5)[0],
            "transposed")
    y.sum().backward()
    assert torch.equal(b.grad, torch.full_like(b, 60.0))
    x0 = torch.zeros(0, 24, device=gpu, requires_grad=True)
    w = torch.ones(24, device=gpu, requires_grad=True)
    y = tg.layer_norm(x0, w)
    dx, dw = torch.autograd.grad(y, (x0, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 24) and torch.equal(dw, torch.zeros_like(w))


def test_layer_norm_constant_rows_and_values_that_are_not_finite(gpu):
    announce("layer norm: constant rows, infinities, NaN")
    x = torch.randn(6, 40, device=gpu)
    x[1] = 3.0
    x[2, 7] = math.nan
    x[4, 0] = math.inf
    y = tg.layer_norm(x)
    assert torch.equal(y[1], torch.zeros(40, device=gpu))
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4]).any())
    rest = [0, 3, 5]
    _within(y[rest], *_norm64(x[rest], None, None, 1e-5)[0], "rows beside them")


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------


def _philox(counter, key):
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _draws(n, seed, offset, first=0):
    out = []
    for group in range(first // 8, -(-(first + n) // 8)):
        words = _philox([group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32],
                        [seed & 0xFFFFFFFF, seed >> 32])
        out += [(w >> s) & 0xFFFF for w in words for s in (0, 16)]
    return np.array(out[first % 8:first % 8 + n])


def test_generator_known_answers():
    """The published known answers of Philox4x32-10."""
    ones = [0xFFFFFFFF] * 4
    assert _philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox(ones, ones[:2]) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert _philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (5, 59), (33, 64), (3, 5, 41)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.93, 1.0])
def test_dropout(gpu, shape, p, dtype):
    announce(f"dropout {shape} p={p} {dtype}")
    n = math.prod(shape)
    seed, offset = 0x9E3779B97F4A7C15 ^ n, (1 << 40) + n
    g = _gen(n)
    x, res = (_rand(g, *shape, dtype=dtype).requires_grad_() for _ in range(2))
    dy = _rand(g, *shape, dtype=dtype)
    t = int(math.floor(p * 65536 + 0.5))
    keep = torch.from_numpy(_draws(n, seed, offset) >= t).to(gpu).view(shape)
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    u, tiny = UNIT[dtype], FLOOR[dtype]
    y = tg.dropout(x, p, seed, offset)
    (dx,) = torch.autograd.grad(y, x, dy)
    for got, src in ((y, x), (dx, dy)):
        want = torch.where(keep, src.detach().double() * scale, 0.0)
        _within(got, want, (u + 3 * U32) * want.abs() + tiny, "dropout")
        assert bool((got[~keep] == 0).all())
    y2 = tg.dropout(x, p, seed, offset, residual=res)
    dx2, dres = torch.autograd.grad(y2, (x, res), dy)
    part = torch.where(keep, x.detach().double() * scale, 0.0)
    want = part + res.detach().double()
    _within(y2, want, u * want.abs() + 3 * U32 * (part.abs() + res.detach().double().abs()) + tiny,
            "residual")
    assert torch.equal(dx2, dx) and torch.equal(dres, dy)
    with torch.no_grad():
        assert torch.equal(tg.dropout(x, p, seed, offset), y)


def test_dropout_layouts_and_alignment(gpu):
    announce("dropout: unaligned and strided inputs give the same mask")
    g = _gen(3)
    base = _rand(g, 4099)
    whole = tg.dropout(base[1:].clone(), 0.3, 11, 5)
    assert torch.equal(tg.dropout(base[1:], 0.3, 11, 5), whole)
    half = tg.dropout(base[1:].clone().to(torch.bfloat16), 0.3, 11, 5)
    assert torch.equal(half == 0, whole == 0)
    m = _rand(g, 40, 64)
    assert torch.equal(tg.dropout(m[:, 3:50], 0.3, 1), tg.dropout(m[:, 3:50].clone(), 0.3, 1))
    assert torch.equal(tg.dropout(m.t(), 0.3, 1), tg.dropout(m.t().clone(), 0.3, 1))
    assert not torch.equal(tg.dropout(m, 0.3, 1, 0), tg.dropout(m, 0.3, 1, 1))
    assert not torch.equal(tg.dropout(m, 0.3, 1, 0), tg.dropout(m, 0.3, 2, 0))
    assert tg.dropout(m[:0], 0.3, 1).shape == (0, 64)


def test_dropout_share_and_dropped_nan(gpu):
    announce("dropout: the share kept, NaN where dropped")
    n, p = 1 << 22, 0.3
    x = torch.ones(n, device=gpu)
    y = tg.dropout(x, p, 1234, 77)
    # a binomial's deviation: six standard deviations
    kept = int((y != 0).sum())
    assert abs(kept - n * (1 - p)) <= 6 * math.sqrt(n * p * (1 - p)) + n * 2.0 ** -17
    x[y == 0] = math.nan
    assert torch.equal(tg.dropout(x, p, 1234, 77), y)


def test_dropout_past_32_bits(gpu):
    """Element indices beyond 2^32, in a tensor of 4.3e9 values."""
    n = (1 << 32) + 77
    announce(f"dropout of {n} bfloat16 values")
    x = torch.ones(n, dtype=torch.bfloat16, device=gpu)
    y = tg.dropout(x, 0.5, 99, 3)
    for first in (0, (1 << 31) - 5, (1 << 32) - 9, n - 101):
        count = min(100, n - first)
        keep = torch.from_numpy(_draws(count, 99, 3, first) >= 32768).to(gpu)
        assert torch.equal(y[first:first + count] != 0, keep), first


# ---------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------

# largest |act'| and |act''|
SLOPE = dict(silu=1.1, gelu=1.13, relu=1.0)
CURVE = dict(silu=0.5, gelu=0.8, relu=0.0)


def _act64(name, g):
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    phi = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def _ffn64(act, x, wg, wu, wd, bg=None, bu=None, bd=None, dy=None):
    """Values and error bounds of y (and dx, dwg, dwu, dwd, dbg, dbu, dbd)."""
    u = UNIT[x.dtype]
    tiny = FLOOR[x.dtype]
    rows, D = x.shape
    F, O = wg.shape[0], wd.shape[0]
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    bg, bu, bd = (zero if t is None else t.double() for t in (bg, bu, bd))

    def product(a, ea, b, eb, k):
        """a @ b of values with errors, k terms, and its error."""
        e = ea @ b.abs() + a.abs() @ eb + ea @ eb + _gamma(k) * (a.abs() @ b.abs())
        return a @ b, e

    def exactly(t):
        return t, torch.zeros_like(t)

    def stored(v, e):
        """Rounded to the tensors' type (float32 keeps 24 bits in either form)."""
        return v, e + (u + U32) * (v.abs() + e) + tiny

    def plus(p, b):
        return p[0] + b, p[1] + U32 * (p[0].abs() + b.abs())

    g, eg = plus(product(*exactly(x), *exactly(wg.t()), D), bg)
    v, ev = plus(product(*exactly(x), *exactly(wu.t()), D), bu)
    a, da = _act64(act, g)
    # the activation's own evaluation: 16 roundings of values no larger than |g| + 1
    ea = SLOPE[act] * eg + 16 * U32 * (a.abs() + U32) + (0 if act == "relu" else 4 * U32 * g.abs())
    h, eh = stored(a * v, ea * v.abs() + a.abs() * ev + ea * ev + 2 * U32 * (a * v).abs())
    y, ey = plus(product(h, eh, *exactly(wd.t()), F), bd)
    out = [stored(y, ey)]
    if dy is None:
        return out
    dy = dy.double()
    dh, edh = product(*exactly(dy), *exactly(wd), O)
    # near a kink the derivative may be either side's
    eda = CURVE[act] * eg + 16 * U32 * (da.abs() + 1) + \
        ((g.abs() <= eg).double() if act == "relu" else 0)
    du, edu = stored(dh * a, edh * a.abs() + (dh.abs() + edh) * ea + 2 * U32 * (dh * a).abs())
    t, et = dh * v, edh * v.abs() + (dh.abs() + edh) * ev + 2 * U32 * (dh * v).abs()
    dg, edg = stored(t * da, et * da.abs() + (t.abs() + et) * eda + 2 * U32 * (t * da).abs())
    p, q = product(dg, edg, *exactly(wg), F), product(du, edu, *exactly(wu), F)
    out.append(stored(p[0] + q[0], p[1] + q[1] + _gamma(F) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())))
    out.append(stored(*product(dg.t(), edg.t(), *exactly(x), rows)))
    out.append(stored(*product(du.t(), edu.t(), *exactly(x), rows)))
    out.append(stored(*product(*exactly(dy.t()), h, eh, rows)))
    for s, es in ((dg, edg), (du, edu), exactly(dy)):
        out.append(stored(s.sum(0), es.sum(0) + _gamma(rows) * s.abs().sum(0)))
    return out


def _ffn_inputs(rows, D, F, O, dtype, bias, seed, pitch=0):
    g = _gen(seed)
    x = _rand(g, rows, D + pitch, dtype=dtype)[:, :D]
    wg, wu = (_rand(g, F, D, dtype=dtype, scale=D ** -0.5) for _ in range(2))
    wd = _rand(g, O, F, dtype=dtype, scale=F ** -0.5)
    b = [_rand(g, n, dtype=dtype, scale=0.3) if bias else None for n in (F, F, O)]
    dy = _rand(g, rows, O + pitch, dtype=dtype, scale=0.5)[:, :O]
    return [x, wg, wu, wd, *b], dy


# (rows, width, hidden, out): one row, fewer than a tile, tiles' edges, odd sizes, wide
FFN_SHAPES = [(1, 1, 1, 1), (1, 64, 256, 48), (2, 3, 5, 2), (16, 16, 32, 3), (17, 8, 40, 16),
              (31, 59, 128, 3), (64, 64, 64, 64), (65, 33, 70, 65), (130, 64, 256, 48),
              (257, 100, 129, 7), (300, 128, 512, 128), (129, 127, 257, 130), (1, 1024, 4096, 1024),
              (9, 520, 1032, 264), (200, 256, 640, 200), (1, 321, 77, 1000), (1031, 48, 96, 48),
              (4099, 64, 128, 3), (600, 1000, 136, 24), (48, 16, 2048, 16)]


def _check_ffn(args, dy, act, what):
    leaves = [None if t is None else t.detach().requires_grad_() for t in args]
    y = tg.gated_ffn(*leaves, activation=act)
    inputs = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, inputs, dy))
    got = [y] + [None if t is None else next(grads) for t in leaves]
    names = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")
    for t, (v, e), name in zip(got, _ffn64(act, *args, dy=dy), names):
        if t is not None:
            assert t.dtype == dy.dtype
            _within(t, v, e, f"{name} of {what}")
    with torch.no_grad():
        assert torch.equal(tg.gated_ffn(*args, activation=act), y)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O", FFN_SHAPES)
def test_gated_ffn(gpu, rows, D, F, O, dtype):
    act = ("silu", "gelu", "relu")[(rows + D) % 3]
    bias = (rows + F) % 2 == 0
    announce(f"gated ffn {rows} x {D}-{F}-{O} {dtype} {act} bias={bias}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, bias, rows + D + F + O)
    _check_ffn(args, dy, act, f"{rows} x {D}-{F}-{O}")


# sums over k split over workgroups (few tiles), 256 x 256 tiles, wavefronts of 32 rows, rows
# that take several passes (hidden values and copies of unaligned rows in parts)
FFN_LARGE = [(70, 264, 4096, 200), (300, 64, 4096, 64), (140, 128, 2048, 100), (33, 1000, 520, 1000),
             (4200, 136, 2048, 136), (15000, 136, 64, 1024), (70001, 64, 40, 48),
             (16500, 136, 4096, 136), ((1 << 20) + 300, 20, 32, 5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O", FFN_LARGE)
def test_gated_ffn_large(gpu, rows, D, F, O, dtype):
    announce(f"gated ffn {rows} x {D}-{F}-{O} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, True, rows + D + F + O)
    _check_ffn(args, dy, "silu", f"{rows} x {D}-{F}-{O}")


# narrow rows whose hidden columns one workgroup holds (65 to 256 of them), every width of its
# exchange, hidden columns that end inside a wavefront's, rows inside a tile, a second pass of rows
FFN_ALONGSIDE = [(35, 64, 65, 64), (64, 64, 128, 33), (1, 32, 96, 3), (1000, 59, 129, 3), (97, 64, 160, 64),
                 (4099, 64, 256, 64), (333, 20, 250, 48), (20001, 32, 256, 32), (66, 33, 224, 64),
                 ((1 << 20) + 300, 12, 100, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,D,F,O", FFN_ALONGSIDE)
def test_gated_ffn_one_workgroup_of_hidden_columns(gpu, rows, D, F, O, act, dtype):
    announce(f"gated ffn {rows} x {D}-{F}-{O} {act} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, F % 2 == 0, rows + D + F + O)
    _check_ffn(args, dy, act, f"{rows} x {D}-{F}-{O}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("pitch", [1, 8, 5])
def test_gated_ffn_pitch_and_activations(gpu, pitch, act, dtype):
    announce(f"gated ffn at a pitch of width + {pitch} {act} {dtype}")
    args, dy = _ffn_inputs(150, 56, 72, 24, dtype, True, pitch, pitch)
    _check_ffn(args, dy, act, f"pitch {pitch}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_ffn_some_gradients(gpu, dtype):
    announce(f"gated ffn: the gradients that are asked for {dtype}")
    args, dy = _ffn_inputs(140, 64, 96, 20, dtype, True, 8)
    whole = _check_ffn(args, dy, "silu", "all")
    for wanted in ((0,), (1,), (3,), (1, 2), (0, 6), (4,), (5, 6)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(args)]
        y = tg.gated_ffn(*leaves)
        got = torch.autograd.grad(y, [leaves[i] for i in wanted], dy)
        for i, t in zip(wanted, got):
            assert torch.equal(t, whole[1 + i]), wanted


def test_gated_ffn_shapes(gpu):
    announce("gated ffn: batch shapes, no rows, weights in other layouts")
    args, dy = _ffn_inputs(30, 24, 40, 6, torch.float32, True, 4)
    y = tg.gated_ffn(*args)
    assert torch.equal(tg.gated_ffn(args[0].reshape(2, 3, 5, 24), *args[1:]), y.view(2, 3, 5, 6))
    one = tg.gated_ffn(args[0][7], *args[1:])
    assert one.shape == (6,)
    _within(one[None], *_ffn64("silu", args[0][7:8], *args[1:])[0], "one row")
    turned = [args[0]] + [t.t().contiguous().t() for t in args[1:4]] + args[4:]
    assert torch.equal(tg.gated_ffn(*turned), y)
    x0 = torch.zeros(0, 24, device=gpu, requires_grad=True)
    leaves = [t.detach().requires_grad_() for t in args[1:]]
    y0 = tg.gated_ffn(x0, *leaves)
    grads = torch.autograd.grad(y0, [x0, *leaves], torch.zeros(0, 6, device=gpu))
    assert y0.shape == (0, 6) and all(bool((t == 0).all()) for t in grads)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_ffn_rows_that_are_not_finite(gpu, dtype):
    """A row's infinities and NaN stay in that row's outputs."""
    announce(f"gated ffn: NaN and infinite rows {dtype}")
    for rows, D, F, O in ((150, 64, 256, 48), (70, 200, 300, 40), (5, 64, 64, 8)):
        args, _ = _ffn_inputs(rows, D, F, O, dtype, True, 6)
        clean = tg.gated_ffn(*args)
        bad = args[0].clone()
        bad[1, 3], bad[4, 0] = math.nan, math.inf
        y = tg.gated_ffn(bad, *args[1:])
        assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[4]).any())
        rest = [i for i in range(rows) if i not in (1, 4)]
        assert torch.equal(y[rest], clean[rest])


def test_gradients_against_differences(gpu):
    """Directional derivatives by central differences of the operators' own forward.  The
    tolerance: the difference quotient's own error, taken from the same quotient in 64 bits,
    the forward's error bound over the step, and the gradients' bounds."""
    announce("gradients against differences")
    step = 2.0 ** -6
    args, dy = _ffn_inputs(37, 20, 50, 9, torch.float32, True, 12)
    for act in ("silu", "gelu"):
        want = _ffn64(act, *args, dy=dy)
        leaves = [t.detach().requires_grad_() for t in args]
        grads = torch.autograd.grad(tg.gated_ffn(*leaves, activation=act), leaves, dy)
        for i, grad in enumerate(grads):
            d = _rand(_gen(i), *args[i].shape, scale=args[i].numel() ** -0.5)
            ends = []
            for sign in (1, -1):
                moved = list(args)
                moved[i] = args[i] + sign * step * d
                ends.append((tg.gated_ffn(*moved, activation=act), _ffn64(act, *moved)[0],
                             (moved[i].double() - args[i].double()) * sign / step))
            along = (ends[0][2] + ends[1][2]) / 2
            quotient, quotient64 = (((a.double() - b.double()) * dy.double()).sum() / (2 * step)
                                    for a, b in ((ends[0][0], ends[1][0]),
                                                 (ends[0][1][0], ends[1][1][0])))
            value, bound = want[1 + i]
            tol = (quotient64 - (value * along).sum()).abs() + (bound * along.abs()).sum() + \
                sum((e[1][1] * dy.double().abs()).sum() for e in ends) / (2 * step)
            assert float((quotient - (grad.double() * along).sum()).abs()) <= float(tol), (act, i)
    x, w, b = (_rand(_gen(k), *s) for k, s in enumerate(((23, 30), (30,), (30,))))
    dy = _rand(_gen(9), 23, 30)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(tg.layer_norm(*leaves), leaves, dy)
    want = _norm64(x, w, b, 1e-5, dy)
    for i, grad in enumerate(grads):
        d = _rand(_gen(i + 5), *leaves[i].shape, scale=leaves[i].numel() ** -0.5)
        ends = []
        for sign in (1, -1):
            moved = [x, w, b]
            moved[i] = moved[i] + sign * step * d
            ends.append((tg.layer_norm(*moved), _norm64(*moved, 1e-5)[0],
                         (moved[i].double() - (x, w, b)[i].double()) * sign / step))
        along = (ends[0][2] + ends[1][2]) / 2
        quotient, quotient64 = (((p.double() - q.double()) * dy.double()).sum() / (2 * step)
                                for p, q in ((ends[0][0], ends[1][0]), (ends[0][1][0], ends[1][1][0])))
        value, bound = want[1 + i]
        tol = (quotient64 - (value * along).sum()).abs() + (bound * along.abs()).sum() + \
            sum((e[1][1] * dy.double().abs()).sum() for e in ends) / (2 * step)
        assert float((quotient - (grad.double() * along).sum()).abs()) <= float(tol), i


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------


def _block(x, w, b, ffn, seed):
    h = tg.layer_norm(x, w, b)
    return tg.dropout(tg.gated_ffn(h, *ffn), 0.2, seed, residual=x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_on_a_side_stream_and_in_a_graph(gpu, dtype):
    announce(f"decoder block on a side stream and in a graph {dtype}")
    args, dy = _ffn_inputs(300, 64, 128, 64, dtype, True, 2)
    x, ffn = args[0], args[1:]
    w, b = torch.ones(64, device=gpu, dtype=dtype), torch.zeros(64, device=gpu, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, *ffn)]

    def step():
        y = _block(*leaves[:3], leaves[3:], 7)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(_rand(_gen(100 + k), 300, 64, dtype=dtype))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, held)), k
        (torch.randn(1 << 20, device=gpu) * 2).sum().item()  # the program's own work between
