"""The decoder operators at the ends of their types' ranges."""
import math

import pytest
import torch

import tidegs_amd as tg
from tests.gpu_util import announce
from tests.test_gpu_decoder_ops import DTYPES, _ffn_inputs

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
