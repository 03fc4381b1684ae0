"""The decoder operators at the ends of their types' ranges, in sums over many rows and
in the kernels that only some sizes reach.

Bounds element by element are those of ``test_gpu_decoder_ops``.  Where a bound over many
rows would admit zeros (it grows with the rows, the sum with their square root), the inputs
leave few terms or the error is taken in the norm, and the test asserts that a sum that
lacks them would not pass.
"""
import math

import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce
from tests.test_gpu_decoder_ops import (DTYPES, UNIT, _act64, _check_ffn, _ffn64, _ffn_inputs, _gen,
                                        _norm64, _rand, _within)

pytestmark = pytest.mark.gpu

NAMES = ("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def _forward_backward(args, dy, act="silu"):
    leaves = [t.detach().requires_grad_() for t in args]
    y = tg.gated_ffn(*leaves, activation=act)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


# up to 32 rows, narrow rows with dx beside the weights' gradients and without, wide rows
FFN_KERNELS = [(5, 64, 64, 8), (150, 64, 256, 48), (150, 128, 80, 100), (70, 200, 300, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O", FFN_KERNELS)
def test_relu_closes_at_minus_infinity(gpu, rows, D, F, O, dtype):
    """A hidden column whose gate's bias is -inf is the column whose gate is zero: relu gives 0
    for both, and no derivative."""
    announce(f"gated ffn: gates at -inf, {rows} x {D}-{F}-{O} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, True, rows)
    closed = torch.arange(F, device=gpu) % 3 == 1
    shut, zero = list(args), list(args)
    shut[4] = args[4].masked_fill(closed, -math.inf)
    zero[4] = args[4].masked_fill(closed, 0)
    zero[1] = args[1].masked_fill(closed[:, None], 0)
    for a, b, name in zip(_forward_backward(shut, dy, "relu"), _forward_backward(zero, dy, "relu"),
                          ("y", *NAMES)):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [59, 64, 1000, 4500])
def test_layer_norm_of_tiny_rows_without_eps(gpu, width, dtype):
    """Rows whose variance, or whose squares, lie below the 32-bit range, beside ordinary ones."""
    announce(f"layer norm without eps, rows from 1 to 2^-100 {width} {dtype}")
    g = _gen(width)
    x = _rand(g, 24, width)
    scale = 2.0 ** -torch.tensor([0, 40, 60, 62, 63, 64, 66, 70, 74, 80, 90, 100], device=gpu)
    x = (x * scale.repeat(2)[:, None]).to(dtype)
    w, b = _rand(g, width, dtype=dtype), _rand(g, width, dtype=dtype)
    dy = _rand(g, 24, width, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = tg.layer_norm(*leaves, 0.0)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    for t, (v, e), name in zip(got, _norm64(x, w, b, 0.0, dy), ("y", "dx", "dw", "db")):
        _within(t, v, e, name)
    # an eps below the squares' range counts as well
    x = _rand(g, 6, width) * 2.0 ** -66
    _within(tg.layer_norm(x, eps=2.0 ** -130), *_norm64(x, None, None, 2.0 ** -130)[0], "with eps")


@pytest.mark.parametrize("scale", [1.0, 1e-2, 1e-6, 3e-7])
@pytest.mark.parametrize("rows,D,F,O", [(20000, 64, 256, 48), (20000, 128, 80, 100),
                                        (20000, 20, 600, 3), (9000, 200, 300, 40)])
def test_half_gradients_of_small_dy(gpu, rows, D, F, O, scale):
    """The weights' gradients of a mean loss: every row's term lies at or below half's smallest
    values, their sums do not.  Each term is rounded to 11 bits twice at most, independently
    of the others, and the sum once: 2^-10 of itself in the norm, and the spacing of half's
    smallest values where the sum is stored."""
    announce(f"half gradients of dy of {scale} {rows} x {D}-{F}-{O}")
    args, dy = _ffn_inputs(rows, D, F, O, torch.float16, True, rows + D)
    dy = (dy.float() * scale).half()
    got = _forward_backward(args, dy)
    for t, (v, _), name in zip(got, _ffn64("silu", *args, dy=dy), ("y", *NAMES)):
        far = (t.double() - v).norm()
        assert float(far) <= 2.0 ** -10 * float(v.norm()) + 2.0 ** -25 * math.sqrt(v.numel()), \
            (name, float(far / v.norm()))


@pytest.mark.parametrize("rows,D,F,O", [(20000, 64, 256, 48), (20000, 128, 80, 100), (9000, 200, 300, 40)])
def test_half_gradients_of_small_hidden_values(gpu, rows, D, F, O):
    """dWd = dy' h of hidden values at half's smallest, and gradients of dy far from it on
    either side: the same bounds."""
    announce(f"half gradients of small hidden values {rows} x {D}-{F}-{O}")
    args, dy = _ffn_inputs(rows, D, F, O, torch.float16, False, rows + D)
    for x_scale, dy_scale in ((1e-3, 1.0), (1e-3, 1e-4), (30.0, 1e-6), (1.0, 100.0)):
        some = [args[0] * x_scale, *args[1:4]]
        leaves = [t.detach().requires_grad_() for t in some]
        d = dy * dy_scale
        grads = torch.autograd.grad(tg.gated_ffn(*leaves), leaves, d)
        for t, (v, _), name in zip(grads, _ffn64("silu", *some, dy=d)[1:], NAMES):
            far = (t.double() - v).norm()
            assert float(far) <= 2.0 ** -10 * float(v.norm()) + 2.0 ** -25 * math.sqrt(v.numel()), \
                (name, x_scale, dy_scale, float(far / v.norm()))


def test_half_gradients_beside_large_rows(gpu):
    """Rows whose x or dy is far larger than the others' leave these as they are without them."""
    announce("half gradients beside large rows")
    for rows, D, F, O in ((300, 64, 256, 48), (300, 128, 80, 100), (300, 200, 300, 40)):
        args, dy = _ffn_inputs(rows, D, F, O, torch.float16, True, 77)
        for k, big in ((0, 3e3), (1, 3e4)):
            x, d = args[0].clone(), dy.clone()
            (x if k == 0 else d)[5] *= big / 4
            got = _forward_backward([x, *args[1:]], d)[1]
            rest = [i for i in range(rows) if i != 5]
            v, e = _ffn64("silu", x[rest], *args[1:], dy=d[rest])[1]
            _within(got[rest], v, e, f"dx beside a row of {big}")


def test_gelu_is_as_near_as_its_formula_in_32_bits(gpu):
    """g Phi(g) and its derivative through a block that passes its gate on, against
    0.5 g (1 + erf(g / sqrt 2)) in 32 bits: no further from 64 bits than 1.5 times that (the
    derivative 2 times: the exponential takes its argument in 32 bits)."""
    announce("gelu against its formula in 32 bits")
    one, zero = torch.ones(1, 1, device=gpu), torch.zeros(1, device=gpu)
    for scale in (0.3, 1.0, 3.0):
        x = _rand(_gen(9), 200000, 1, scale=scale).requires_grad_()
        y = tg.gated_ffn(x, one, one * 0, one, zero, zero + 1, zero, activation="gelu")
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        g = x.detach()
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        slope = phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        for got, plain, want, times in zip((y.detach(), dx), (g * phi, slope), _act64("gelu", g.double()),
                                           (1.5, 2.0)):
            far, plain_far = (float((t.double() - want).norm()) for t in (got, plain))
            assert far <= times * plain_far, (scale, far, plain_far)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_open_and_large_gates(gpu, act, dtype):
    """A gate of +inf gives an infinity, large ones their own value or 0."""
    announce(f"gated ffn: gates of +inf and large ones {act} {dtype}")
    for rows in (5, 50):
        for D in (8, 200):
            x = torch.zeros(rows, D, dtype=dtype, device=gpu)
            w = torch.zeros(3, D, dtype=dtype, device=gpu)
            one = torch.ones(3, dtype=dtype, device=gpu)
            for gate, want in ((math.inf, math.inf), (30000.0, 30000.0), (200.0, 200.0), (-200.0, 0.0),
                               (-30000.0, 0.0)):
                wd = torch.tensor([[1.0, 0.0, 0.0]], dtype=dtype, device=gpu)
                bg = torch.tensor([gate, 0, 0], dtype=dtype, device=gpu)
                y = tg.gated_ffn(x, w, w, wd, bg, one, None, activation=act)
                assert torch.equal(y, torch.full_like(y, want)), (rows, D, gate, y.flatten()[0])


@pytest.mark.parametrize("rows,O", [(32, 128), (1000, 128), (500, 300)])
def test_float32_products_of_computed_values(gpu, rows, O):
    """A hidden value times a weight, one product, where the parts that its six products of
    bfloat16 planes leave out are largest: 2^-24 of it at most, and a last bit of the sum."""
    announce(f"float32 products of hidden values {rows} x {O}")
    g = _gen(rows)
    x = 1 + 2.0 ** -7 * torch.rand(rows, 1, generator=g, device=gpu)
    wd = 1 + 2.0 ** -7 * torch.rand(O, 1, generator=g, device=gpu)
    one, zero = torch.ones(1, 1, device=gpu), torch.zeros(1, device=gpu)
    y = tg.gated_ffn(x, one, 0 * one, wd, zero, zero + 1, None, activation="relu")
    want = x.double() * wd.double().t()
    assert float(((y.double() - want) / want).abs().max()) <= 2.0 ** -24 + 2.0 ** -23


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,F,O", [(5, 8, 3, 4), (50, 8, 3, 4), (66000, 8, 40, 4), (50, 100, 70, 20),
                                        (300, 64, 100, 33), (300, 33, 130, 64), (50, 64, 2100, 7),
                                        (50, 200, 70, 20)])
def test_infinite_rows_come_out_infinite(gpu, rows, D, F, O, dtype):
    """Weights and rows are positive, so a row with an infinity has infinite outputs, whatever
    the hidden columns are padded to; so has a row's dx where dy has one."""
    announce(f"gated ffn: infinite rows {rows} x {D}-{F}-{O} {dtype}")
    g = _gen(F)
    args = [torch.rand(s, generator=g, device=gpu).add(0.5).to(dtype)
            for s in ((rows, D), (F, D), (F, D), (O, F), (F,), (F,), (O,))]
    args[1:4] = [w / w.shape[1] for w in args[1:4]]
    dy = torch.rand(rows, O, generator=g, device=gpu).to(dtype)
    clean = _forward_backward(args, dy)[:2]
    bad, dbad = args[0].clone(), dy.clone()
    bad[3, D - 1], dbad[4, 0] = math.inf, math.inf
    with torch.no_grad():
        y = tg.gated_ffn(bad, *args[1:])
    dx = _forward_backward(args, dbad)[1]
    for t, row, c in ((y, 3, clean[0]), (dx, 4, clean[1])):
        assert bool((t[row] == math.inf).all()), t[row]
        rest = torch.arange(rows, device=gpu) != row
        assert torch.equal(t[rest], c[rest])


# rows in several passes: narrow rows with dx beside the weights' gradients and without, wide
# rows; the first and the last pass's rows
FFN_PASSES = [((1 << 20) + 300, 20, 32, 5, 1 << 20), ((1 << 20) + 300, 12, 100, 7, 1 << 20),
              (16500, 136, 4096, 136, 16384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O,one_pass", FFN_PASSES)
def test_every_pass_reaches_the_sums_over_rows(gpu, rows, D, F, O, one_pass, dtype):
    """dy is zero but in some rows of one pass: the sums are those rows', which a bound over
    them alone checks.  Zeros, all that is left without that pass, lie outside it."""
    announce(f"gated ffn: passes of {rows} x {D}-{F}-{O} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, True, rows + F)
    for first, last in ((0, 100), (one_pass - 100, one_pass), (one_pass, one_pass + 100),
                        (rows - 100, rows)):
        some = torch.zeros_like(dy)
        some[first:last] = dy[first:last]
        got = _forward_backward(args, some)
        want = _ffn64("silu", args[0][first:last].contiguous(), *args[1:], dy=dy[first:last])
        for k, name in enumerate(NAMES):
            v, e = want[1 + k]
            t = got[1 + k]
            if name == "dx":
                assert not bool(t[:first].any()) and not bool(t[last:].any())
                t = t[first:last]
            else:
                assert float((v.abs() > e).double().mean()) > 0.7, f"{name}: zeros would pass"
            _within(t, v, e, f"{name} of rows {first}:{last}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O", [(70001, 64, 40, 48), ((1 << 20) + 30000, 20, 32, 5),
                                        ((1 << 20) + 30000, 12, 100, 7), (40001, 100, 64, 90),
                                        (18000, 136, 4096, 136)])
def test_sums_over_many_rows(gpu, rows, D, F, O, dtype):
    """The parameters' gradients in the norm.  A row's terms carry two independent roundings of
    the tensors' type and the sum one: 3 u of the whole; of float32, whose terms carry some tens
    of 2^-24 and whose partial sums are of up to 2^17 rows, 2^-17.  A pass that is left out
    or zeros are further off."""
    announce(f"gated ffn: sums over {rows} rows {D}-{F}-{O} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, True, rows + F + 1)
    got = _forward_backward(args, dy)
    want = _ffn64("silu", *args, dy=dy)
    part = (1 << 20) if rows > 1 << 20 else 16384
    lost = _ffn64("silu", args[0][:part].contiguous(), *args[1:], dy=dy[:part]) if part < rows else None
    limit = 2.0 ** -17 if dtype == torch.float32 else 3 * UNIT[dtype]
    for k in range(2, 8):
        v = want[k][0]
        assert float((got[k].double() - v).norm() / v.norm()) <= limit, NAMES[k - 1]
        if lost is not None:
            assert float((lost[k][0] - v).norm() / v.norm()) > 2 * limit, NAMES[k - 1]


# up to 32 rows with 16 outputs a workgroup (from 2048 outputs on); 16-bit rows 32 a wavefront
# (from 65536 rows on) in the widest dx kernels and in the forward's, by their outputs
FFN_BRANCHES = [(1, 64, 64, 2048), (32, 64, 64, 2051), (32, 64, 64, 2048), (1, 70, 33, 2051),
                (66000, 128, 48, 128), (66000, 100, 40, 20), (66000, 64, 48, 32), (66000, 64, 48, 64),
                (66000, 40, 48, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,F,O", FFN_BRANCHES)
def test_kernels_of_some_sizes(gpu, rows, D, F, O, dtype):
    announce(f"gated ffn {rows} x {D}-{F}-{O} {dtype}")
    args, dy = _ffn_inputs(rows, D, F, O, dtype, True, rows + D + F + O)
    _check_ffn(args, dy, "silu", f"{rows} x {D}-{F}-{O}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 16, 17, 32])
@pytest.mark.parametrize("D,F,O", [(64, 256, 48), (100, 1000, 30), (256, 1024, 2051)])
def test_few_rows_keep_their_hidden_values(gpu, rows, D, F, O, dtype):
    """Up to 32 rows multiply a hidden value with what its rounding left.  What is lost then, u^2
    of a hidden value and the sums' 2^-24 sqrt(F), is a hundredth of the results' spacing at most,
    so y is the 64-bit result rounded but for one value in fifty (and two); hidden values rounded
    once move one in ten at least."""
    announce(f"gated ffn: hidden values of {rows} rows {D}-{F}-{O} {dtype}")
    args, _ = _ffn_inputs(rows, D, F, O, dtype, True, rows + F)
    x, wg, wu, wd, bg, bu, bd = (t.double() for t in args)
    h = _act64("silu", x @ wg.t() + bg)[0] * (x @ wu.t() + bu)
    want = (h @ wd.t() + bd).to(dtype)
    once = (h.to(dtype).double() @ wd.t() + bd).to(dtype)
    n = want.numel()
    assert int((once != want).sum()) > 2 + n / 10, "a hidden value rounded once would pass"
    assert int((tg.gated_ffn(*args) != want).sum()) <= 2 + n / 50


def test_half_hidden_values_up_to_the_largest(gpu):
    """A hidden value of 65472 is half's own; its product with a small weight is right."""
    announce("gated ffn: half hidden values near the largest")
    for rows, D, F, O in ((5, 64, 64, 8), (150, 64, 64, 48), (150, 200, 300, 40)):
        one = torch.zeros(F, D, dtype=torch.float16, device=gpu)
        one[:, 0] = 1
        x = torch.zeros(rows, D, dtype=torch.float16, device=gpu)
        x[:, 0] = 255.875  # squared 65472.0156: rounds to 65472
        wd = torch.zeros(O, F, dtype=torch.float16, device=gpu)
        wd[:, 1] = 2.0 ** -6
        y = tg.gated_ffn(x, one, one, wd, activation="relu")
        assert torch.equal(y, torch.full_like(y, 1023.0)), y.flatten()[0]


def test_more_than_a_billion_rows(gpu):
    """2^30 + 100 rows of one value: four threads a row pass what one launch may have."""
    rows, part = (1 << 30) + 100, 1000
    announce(f"gated ffn: {rows} rows of one value")
    g = _gen(30)
    x = torch.empty(rows, 1, device=gpu).uniform_(-2, 2, generator=g).requires_grad_()
    args = [torch.tensor(v, device=gpu).view(s) for v, s in ((0.75, (1, 1)), (-0.5, (1, 1)), (2.0, (1, 1)),
                                                             (0.25, (1,)), (0.5, (1,)), (-1.0, (1,)))]
    y = tg.gated_ffn(x, *args)
    dy = torch.empty(rows, 1, device=gpu).uniform_(-1, 1, generator=g)
    (dx,) = torch.autograd.grad(y, x, dy)
    for first in (0, (1 << 29) - 500, (1 << 30) - 500, rows - part):
        some = slice(first, first + part)
        for t, (v, e) in zip((y, dx), _ffn64("silu", x.detach()[some], *args, dy=dy[some])):
            _within(t[some], v, e, f"rows from {first}")
