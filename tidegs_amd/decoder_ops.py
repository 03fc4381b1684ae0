"""Operators of a decoder over per-Gaussian features or rendered images of them:
``layer_norm``, ``group_norm``, ``dropout`` and ``gated_ffn``, forward and backward in the HIP
kernels of ``libtidegs_amd.so``.

TideGS itself stores SH coefficients with every Gaussian; these are what a small
network needs that computes colours (or corrections of them) from features
stored there and from an embedding of the image.  Inputs are float32, bfloat16 or
float16 GPU tensors of ``[..., width]``; sums are taken in 32 bits or more and a
result is rounded once, to its tensor's type.  A dense tensor, or a matrix of dense
rows at one pitch (columns of a resident table), is read in place by ``layer_norm``,
``group_norm`` and ``gated_ffn``, a dense one by ``dropout``; any other is copied first.  Every call
runs on the current stream, takes its workspaces from torch's allocator and gives the
same bits for the same inputs.  Gradients are taken in reverse mode, once: a tangent of
forward mode or a second derivative raises.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_MAX_WIDTH = 65536


def _dtype(x: Tensor, name: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    return code


def _on_gpu(x: Tensor, name: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(
            f"{name} must be a GPU tensor (the TideGS HIP kernels have no CPU path)")


def _rows(x: Tensor):
    """``x`` as rows of its last dimension: (tensor, rows, pitch), in place where its
    rows lie at one pitch."""
    width = x.shape[-1]
    if x.is_contiguous():
        return x, (x.numel() // width if width else 0), width
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= width:
        return x, x.shape[0], x.stride(0)
    x = x.contiguous()
    return x, (x.numel() // width if width else 0), width


def _parameter(t: Optional[Tensor], name: str, shape, x: Tensor, also=()) -> Optional[Tensor]:
    """A weight or bias: its shape, type and device checked, dense."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != x.dtype and t.dtype not in also:
        raise TypeError(f"{name} must be {x.dtype} like x, got {t.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=1024)
def _workspace_size(query: str, *sizes: int) -> int:
    return getattr(N.load(), query)(*sizes)


def _recorded(*tensors: Optional[Tensor]) -> bool:
    """Whether a call goes through its autograd Function: a gradient is asked for, or a tensor
    carries a tangent, which the Function refuses (the operators have no forward mode) and
    the bare call would lose."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:  # (asked first: unpacking costs a quarter us a tensor)
        return any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                   for t in tensors)
    return False


def _once(backward):
    """``backward`` as an autograd Function's: not differentiable again, which only a
    backward that records its own graph has to be told (the wrapper that tells it
    costs as much as a launch)."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, dy):
        return recorded(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)

    return staticmethod(run)


# ---------------------------------------------------------------------------
# layer_norm
# ---------------------------------------------------------------------------


def _layer_norm_fwd(x, weight, bias, eps):
    """(x as it is read, y, the arguments that the backward's call shares)."""
    x, rows, pitch = _rows(x)
    width = x.shape[-1]
    y = x.new_empty(x.shape)
    code = _DTYPES[x.dtype]
    w = weight if weight is not None else bias
    w_code = code if w is None or w.dtype == x.dtype else _DTYPES[w.dtype]
    N.call("tgs_layer_norm_fwd", rows, width, code, x.data_ptr(), pitch, N.ptr(weight),
           N.ptr(bias), w_code, eps, y.data_ptr(), N.stream_handle(x.device))
    return x, y, (rows, width, code, pitch, w_code, eps)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, y, ctx.call = _layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias)
        return y

    @_once
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        rows, width, code, pitch, w_code, eps = ctx.call
        dy_pitch = width
        if not dy.is_contiguous():
            dy, _, dy_pitch = _rows(dy)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = dw = db = ws = None
        ws_bytes = 0
        if need_x:
            dx = x.new_empty(x.shape)
        if need_w:
            dw = weight.new_empty(width)
        if need_b:
            db = bias.new_empty(width)
        if need_w or need_b:
            ws_bytes = _workspace_size("tgs_layer_norm_bwd_workspace_size", rows, width)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
        N.call("tgs_layer_norm_bwd", rows, width, code, x.data_ptr(), pitch, dy.data_ptr(),
               dy_pitch, N.ptr(weight), w_code, eps, N.ptr(dx), N.ptr(dw), N.ptr(db), N.ptr(ws),
               ws_bytes, N.stream_handle(x.device))
        return dx, dw, db, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    x [..., width]; weight and bias [width] of x's type, or both float32, or
    None.  Differentiable in all three.
    """
    _dtype(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x needs a last dimension to normalise, got shape {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    _on_gpu(x, "x")
    shape = x.shape[-1:]
    weight = _parameter(weight, "weight", shape, x, (torch.float32,))
    bias = _parameter(bias, "bias", shape, x, (torch.float32,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: one type is needed")
    if _recorded(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _layer_norm_fwd(x, weight, bias, float(eps))[1]


# ---------------------------------------------------------------------------
# group_norm
# ---------------------------------------------------------------------------

_MIN_EPS, _MAX_EPS = 2.0 ** -80, 2.0 ** 80


_node = None


def _group_norm_node():
    """The module that has group norm's node of the autograd graph (built with the library): both
    directions of few values take 65 us a call, as a Function in Python they took 107."""
    global _node
    if _node is None:
        lib = N.load()
        from . import _group_norm_node as node

        names = ("last_error", "group_norm_stats_size", "group_norm_fwd_workspace_size",
                 "group_norm_fwd", "group_norm_bwd_workspace_size", "group_norm_bwd")
        node.bind(*(ctypes.cast(getattr(lib, "tgs_" + name), ctypes.c_void_p).value
                    for name in names))
        _node = node
    return _node


def group_norm(x: Tensor, num_groups: int, weight: Optional[Tensor] = None,
               bias: Optional[Tensor] = None, eps: float = 1e-5,
               activation: Optional[str] = None) -> Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` with mean and variance over each
    sample's groups of channels.

    x [samples, ..., width], channels last, as ``rasterize_to_pixels`` leaves images; a group is
    width / num_groups neighbouring channels of all of a sample's pixels.  weight and bias
    [width] of x's type, or both float32, or None; ``activation`` None, "silu", "gelu" (with the
    error function) or "relu".  Differentiable in all three tensors.  Images whose pixels lie at
    one pitch (columns of wider rows) are read in place.  A NaN or an infinity makes its
    sample's group NaN and no other, and so do differences past 1e18, whose squares leave
    float32.  A backward is captured only while no eager graph of the default stream holds the
    tensors it gives gradients to: it raises otherwise.
    """
    _dtype(x, "x")
    act = 3 if activation is None else _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be None or one of {sorted(_ACTIVATIONS)}, "
                         f"got {activation!r}")
    if x.dim() < 2 or not 0 < x.shape[-1] <= _MAX_WIDTH:
        raise ValueError(f"x needs samples and 1..{_MAX_WIDTH} channels, got shape "
                         f"{tuple(x.shape)}")
    if num_groups < 1 or x.shape[-1] % num_groups:
        raise ValueError(f"{x.shape[-1]} channels do not make {num_groups} groups")
    if not _MIN_EPS <= eps <= _MAX_EPS:
        raise ValueError(f"eps must lie in {_MIN_EPS:.3g}..{_MAX_EPS:.3g} (squares below leave "
                         f"float32), got {eps}")
    _on_gpu(x, "x")
    shape = x.shape[-1:]
    weight = _parameter(weight, "weight", shape, x, (torch.float32,))
    bias = _parameter(bias, "bias", shape, x, (torch.float32,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: one type is needed")
    return _group_norm_node().group_norm(x, weight, bias, int(num_groups), float(eps), act,
                                         _recorded(x, weight, bias))


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------


def _dropout(x, residual, threshold, seed, offset):
    y = torch.empty_like(x)
    N.call("tgs_dropout", x.numel(), _DTYPES[x.dtype], x.data_ptr(), N.ptr(residual),
           y.data_ptr(), threshold, seed, offset, N.stream_handle(x.device))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset):
        ctx.draws = threshold, seed, offset
        return _dropout(x, residual, threshold, seed, offset)

    @_once
    def backward(ctx, dy):
        dx = _dropout(dy.contiguous(), None, *ctx.draws) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: Tensor, p: float, seed: int, offset: int = 0,
            residual: Optional[Tensor] = None) -> Tensor:
    """``x`` with a share ``p`` of its values set to zero and the rest scaled by
    1 / (1 - p), plus ``residual`` if given.

    Which values stay is a function of ``seed`` (a run's or a layer's), ``offset``
    (a step's) and a value's index in ``x`` alone: the mask is not stored, the
    backward computes it again, and the same three give the same mask for every
    element type.  p is taken to the nearest 1/65536, and the scale is that
    share's.  A dropped value is not read into the result (a NaN there gives
    0), and p = 1 drops all.  For evaluation leave the call out.
    """
    _dtype(x, "x")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must lie in [0, 1], got {p}")
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise ValueError(f"seed and offset must be unsigned 64-bit integers, got {seed}, {offset}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("residual must have x's shape, type and device")
    _on_gpu(x, "x")
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    threshold = int(math.floor(p * 65536 + 0.5))
    if _recorded(x, residual):
        return _Dropout.apply(x, residual, threshold, int(seed), int(offset))
    return _dropout(x, residual, threshold, int(seed), int(offset))


# ---------------------------------------------------------------------------
# gated_ffn
# ---------------------------------------------------------------------------


def _gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
    """(x as it is read, y, the arguments that the backward's call shares)."""
    x, rows, pitch = _rows(x)
    (hidden, width), out = w_gate.shape, w_down.shape[0]
    y = x.new_empty((*x.shape[:-1], out))
    code = _DTYPES[x.dtype]
    nbytes = _workspace_size("tgs_gated_ffn_fwd_workspace_size", rows, width, hidden, out, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    N.call("tgs_gated_ffn_fwd", rows, width, hidden, out, code, act, x.data_ptr(), pitch,
           w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), N.ptr(b_gate), N.ptr(b_up),
           N.ptr(b_down), y.data_ptr(), ws.data_ptr(), nbytes, N.stream_handle(x.device))
    return x, y, (rows, width, hidden, out, code, act, pitch)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
        x, y, ctx.call = _gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)
        ctx.save_for_backward(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
        return y

    @_once
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        x, w_gate, w_up, w_down, b_gate, b_up, _ = saved
        rows, width, hidden, out, code, act, pitch = ctx.call
        dy_pitch = out
        if not dy.is_contiguous():
            dy, _, dy_pitch = _rows(dy)
        grads = [t.new_empty(t.shape) if need else None
                 for t, need in zip(saved, ctx.needs_input_grad)]
        nbytes = _workspace_size("tgs_gated_ffn_bwd_workspace_size", rows, width, hidden, out,
                                 code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        N.call("tgs_gated_ffn_bwd", rows, width, hidden, out, code, act, x.data_ptr(), pitch,
               w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), N.ptr(b_gate), N.ptr(b_up),
               dy.data_ptr(), dy_pitch, *map(N.ptr, grads), ws.data_ptr(), nbytes,
               N.stream_handle(x.device))
        return *grads, None


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
              b_gate: Optional[Tensor] = None, b_up: Optional[Tensor] = None,
              b_down: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``(act(x w_gate' + b_gate) * (x w_up' + b_up)) w_down' + b_down``.

    x [..., width], w_gate and w_up [hidden, width], w_down [out, hidden], biases
    [hidden], [hidden], [out] or None, all of one type; ``activation`` "silu",
    "gelu" (with the error function) or "relu".  Returns [..., out].
    Differentiable in every tensor; the backward computes the hidden values
    again.  The hidden product and its gradients are rounded to the tensors'
    type between the matrix products, as a stored hidden tensor would be
    (float32 tensors are not, nor is the hidden product of up to 32 rows: a row's last
    bits depend on which side of 32 its call is).  Half
    precision's backward scales them to the type's range first, by powers of two, so
    that sums over rows of gradients below its smallest values come out; a hidden
    product past 65504, or a gradient of one, is infinite there.  A row's infinities
    and NaN stay in that row's y and dx; in float32 an infinity comes out as NaN.
    """
    _dtype(x, "x")
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if x.dim() == 0 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError("x needs a last dimension and the weights two")
    hidden, width, out = w_gate.shape[0], x.shape[-1], w_down.shape[0]
    if not all(0 < n <= _MAX_WIDTH for n in (hidden, width, out)):
        raise ValueError(f"width, hidden and out must lie in 1..{_MAX_WIDTH}, got "
                         f"{width}, {hidden}, {out}")
    _on_gpu(x, "x")
    w_gate = _parameter(w_gate, "w_gate", (hidden, width), x)
    w_up = _parameter(w_up, "w_up", (hidden, width), x)
    w_down = _parameter(w_down, "w_down", (out, hidden), x)
    b_gate = _parameter(b_gate, "b_gate", (hidden,), x)
    b_up = _parameter(b_up, "b_up", (hidden,), x)
    b_down = _parameter(b_down, "b_down", (out,), x)
    args = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if _recorded(*args):
        return _GatedFfn.apply(*args, act)
    return _gated_ffn_fwd(*args, act)[1]
