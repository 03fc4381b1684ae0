"""The step over all tensors of a network at once: ``adamw_step`` and ``grad_norm``, and the
optimizer ``AdamW`` that calls them, in the HIP kernels of ``libtidegs_amd.so``.

``GPUResidentAdam`` updates the touched rows of resident blocks; this is for everything else
that is trained beside them (a decoder's parameters, features, whole tables).  One launch takes
up to 56 tensors of float32, bfloat16 or float16, whatever their sizes and alignment.  States
are float32, or 8 bits a value and a scale for each 128 of them: the first moment float8_e4m3fn to
nearest, the second float8_e5m2 rounded stochastically (it moves by a thousandth a step, which
nearest rounding would lose).  16-bit parameters are rounded stochastically, too.  The draws
follow from the seed, the step, a tensor's number and a value's index alone, so the same
calls give the same bits.  Every call runs on the current stream.
"""
from __future__ import annotations

import array
import itertools
import math
import struct
from typing import Iterable, Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _native as N
from .decoder_ops import _DTYPES, _workspace_size

_BLOCK = 128
_KEYS = {32: ("exp_avg", "exp_avg_sq"),
         8: ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
_STATES = {32: (torch.float32, torch.float32), 8: (torch.float8_e4m3fn, torch.float8_e5m2)}

_reader = None


def _lists():
    """The module that reads lists of tensors (built with the library)."""
    global _reader
    if _reader is None:
        N.load()  # (first: its error says how to build both)
        from . import _tensor_lists as _reader
    return _reader


def _on_one_gpu(tensors: Sequence[Tensor], name: str) -> torch.device:
    devices = {t.device for t in tensors}
    if len(devices) > 1:
        raise ValueError(f"{name} must be on one device, got {sorted(map(str, devices))}")
    device = devices.pop()
    if device.type != "cuda":
        raise RuntimeError(
            f"{name} must be GPU tensors (the TideGS HIP kernels have no CPU path)")
    return device


# ---------------------------------------------------------------------------
# grad_norm
# ---------------------------------------------------------------------------


def grad_norm(tensors: Iterable[Tensor]) -> Tensor:
    """The 2-norm of all values of all ``tensors`` together, a float32 tensor without
    dimensions.

    Squares are summed in 64 bits and in a fixed order; tensors of float32, bfloat16 and
    float16 may be mixed.  An infinity or a NaN anywhere comes out.
    """
    tensors = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    if not tensors:
        raise ValueError("grad_norm needs a tensor at least")
    found = _lists().spans(tensors)
    if found is None:  # not all contiguous, or something is wrong
        for t in tensors:
            if t.dtype not in _DTYPES:
                raise TypeError(f"tensors must be float32, bfloat16 or float16, got {t.dtype}")
        device = _on_one_gpu(tensors, "tensors")
        tensors = [t if _is_dense(t) else t.contiguous() for t in tensors]
        rows = array.array("Q", itertools.chain.from_iterable(
            (t.data_ptr(), t.numel(), _DTYPES[t.dtype]) for t in tensors)).tobytes()
    else:
        device, rows = tensors[0].device, found[1]
    norm = torch.empty((), dtype=torch.float32, device=device)
    nbytes = _workspace_size("tgs_grad_norm_workspace_size", len(tensors))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    N.launch(device, "tgs_grad_norm", len(tensors), rows, norm.data_ptr(), ws.data_ptr(), nbytes)
    return norm


def _is_dense(t: Tensor) -> bool:
    """Whether the values fill a range of memory, each place once, in any order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


# ---------------------------------------------------------------------------
# adamw_step
# ---------------------------------------------------------------------------


def _check_hyper(lr, betas, eps, weight_decay) -> None:
    if not (math.isfinite(lr) and lr >= 0):
        raise ValueError(f"lr must not be negative, got {lr}")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"betas must lie in [0, 1), got {tuple(betas)}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must not be negative, got {eps}")
    if not (math.isfinite(weight_decay) and weight_decay >= 0):
        raise ValueError(f"weight_decay must not be negative, got {weight_decay}")


def _check_seed(seed: int) -> int:
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must be an unsigned 64-bit integer, got {seed}")
    return int(seed)


_GROUP = struct.Struct("5d3Q")  # tgs_adamw_group


class _Call:
    """The arguments of one ``tgs_adamw``: tensors, checked, and their groups."""

    def __init__(self, bits: int):
        self.bits = bits
        self.groups = b""
        self.n_groups = 0

    def group(self, lr, betas, eps, weight_decay, step=0, lr_device=None, step_device=None) -> int:
        self.groups += _GROUP.pack(lr, *betas, eps, weight_decay, step, N.ptr(lr_device) or 0,
                                   N.ptr(step_device) or 0)
        self.n_groups += 1
        return self.n_groups - 1

    def check(self, p, g, m, v, m_scale, v_scale):
        """One parameter's tensors; the gradient as it is read."""
        if p.dtype not in _DTYPES:
            raise TypeError(f"parameters must be float32, bfloat16 or float16, got {p.dtype}")
        shape, device = p.shape, p.device
        if g.layout is not torch.strided:
            raise RuntimeError("sparse gradients are not taken")
        if g.shape != shape or g.dtype != p.dtype or g.device != device:
            raise ValueError(f"a gradient must have its parameter's shape, type and device "
                             f"({tuple(shape)}, {p.dtype}, {device}), got {tuple(g.shape)}, "
                             f"{g.dtype}, {g.device}")
        types = _STATES[self.bits]
        for t, dtype, name in ((m, types[0], "exp_avg"), (v, types[1], "exp_avg_sq")):
            if t.shape != shape or t.dtype != dtype or t.device != device:
                raise ValueError(f"{name} must have its parameter's shape and device and be {dtype}, "
                                 f"got {tuple(t.shape)}, {t.dtype}, {t.device}")
        if self.bits == 8:
            blocks = (p.numel() + _BLOCK - 1) // _BLOCK
            for t, name in ((m_scale, "exp_avg_scale"), (v_scale, "exp_avg_sq_scale")):
                if t.shape != (blocks,) or t.dtype != torch.float32 or t.device != device \
                        or not t.is_contiguous():
                    raise ValueError(f"{name} must hold {blocks} float32 values on {device}, one "
                                     f"for each {_BLOCK}")
        if p.is_contiguous() and m.is_contiguous() and v.is_contiguous():
            return g.contiguous()
        if not (_is_dense(p) and m.stride() == p.stride() and v.stride() == p.stride()):
            raise ValueError("parameters and states must be dense, in one order of their values")
        return g if g.stride() == p.stride() else torch.empty_like(p).copy_(g)

    def checked(self, params, grads, states, numbers, of):
        """(gradients as they are read, rows of tgs_adamw_tensor) with every tensor checked: what is
        wrong raises, what is merely not contiguous is taken as ``check`` does."""
        none = (itertools.repeat(None),) * (4 - len(states))
        grads = [self.check(*t) for t in zip(params, grads, *states, *none)]
        _on_one_gpu(params, "parameters")
        rows, written = array.array("Q"), []
        for k, p in enumerate(params):
            at = [t[k].data_ptr() for t in (params, *states)]
            if p.numel():
                written += at
            rows.extend((at[0], grads[k].data_ptr(), *at[1:], *(0,) * (4 - len(states)), p.numel(),
                         numbers[k] | of[k] << 32, _DTYPES[p.dtype]))
        if len(set(written)) != len(written):
            raise ValueError("a parameter or a state is there twice")
        return grads, rows.tobytes()

    def run(self, params, grads, states, numbers, of, seed, norm, max_norm, live=False) -> None:
        """``states``: exp_avgs, exp_avg_sqs and, of 8 bits, both lists of scales; ``of``: the
        group of each parameter."""
        n = len(params)
        if not n:
            return
        scales = states[2:] or (None, None)
        found = _lists().adamw(params, grads, *states[:2], *scales, _BLOCK, numbers, of)
        if found is None:
            grads, rows = self.checked(params, grads, states, numbers, of)
        else:
            rows = found[1]
        device = params[0].device
        if norm is not None and (norm.numel() != 1 or norm.dtype != torch.float32
                                 or norm.device != device):
            raise ValueError("grad_norm must be one float32 value on the parameters' device")
        ws, nbytes = None, 0
        if live:
            nbytes = _workspace_size("tgs_adamw_workspace_size", self.n_groups)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        N.launch(device, "tgs_adamw", n, rows, self.n_groups, self.groups, self.bits, seed,
                 N.ptr(norm), max_norm, N.ptr(ws), nbytes)
        increment_version(params)


def _check_max_norm(max_norm) -> float:
    if not max_norm > 0:
        raise ValueError(f"max_norm must be positive, got {max_norm}")
    return float(max_norm)


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], step: int, *, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, exp_avg_scales: Optional[Sequence[Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[Tensor]] = None,
               grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None,
               seed: int = 0) -> None:
    """Step number ``step`` (from 1) of AdamW on ``params``, in place, with its states.

    With g the gradient, times min(1, max_norm / (grad_norm + 1e-6)) where both are
    given (``grad_norm`` as the function of that name returns it, which stays on the GPU)::

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    A gradient has its parameter's type.  Without scales the states are float32, of the
    parameters' shapes.  With them (float32, ceil(n / 128) of a parameter of n values, in the
    order of memory) exp_avg is float8_e4m3fn and exp_avg_sq float8_e5m2, to be multiplied by
    their block's scale; zeros are a start for all four.  What is rounded stochastically (exp_avg_sq
    of 8 bits, parameters of 16) draws from ``seed``, the step, a tensor's place in the lists and
    a value's index.  Parameters and states are dense and do not overlap; a gradient in another
    order is copied.  A NaN stays in its value, and an infinity, too: the rest of the block is
    not touched by it.
    """
    bits = 32 if exp_avg_scales is None else 8
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise ValueError("both states have scales, or none")
    lists = [params, grads, exp_avgs, exp_avg_sqs]
    lists += [exp_avg_scales, exp_avg_sq_scales] if bits == 8 else []
    if len({len(t) for t in lists}) != 1:
        raise ValueError(f"lists of one length are needed, got {[len(t) for t in lists]}")
    _check_hyper(lr, betas, eps, weight_decay)
    if not 1 <= step < 1 << 32:
        raise ValueError(f"steps count from 1, below 2^32: got {step}")
    if (grad_norm is None) != (max_norm is None):
        raise ValueError("grad_norm and max_norm go together")
    max_norm = 0.0 if max_norm is None else _check_max_norm(max_norm)
    call = _Call(bits)
    call.group(lr, betas, eps, weight_decay, step)
    n = len(params)
    call.run(*lists[:2], lists[2:], range(n), [0] * n, _check_seed(seed), grad_norm, max_norm)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------


class AdamW(torch.optim.Optimizer):
    """AdamW whose whole step is a launch for every 56 tensors of a type.

    ``state_bits`` is 32 or 8 (see ``adamw_step``).  ``step(max_norm=...)`` clips the
    gradients by their common norm on the way, without writing them; ``last_norm`` is that
    norm, on the GPU.  A parameter without a gradient is left out of a step and keeps its
    own count of steps.

    ``capturable=True`` counts steps on the GPU, one count for each parameter group, so that a
    captured step counts its replays; its learning rates may be float32 GPU tensors, read at
    every step.  Step once before the capture: states are not made within one.
    """

    def __init__(self, params, lr=1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 seed: int = 0, capturable: bool = False):
        if state_bits not in _STATES:
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        self.state_bits, self.seed, self.capturable = state_bits, _check_seed(seed), capturable
        self.last_norm: Optional[Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group) -> None:
        group = {**self.defaults, **param_group}
        self._lr(group)
        _check_hyper(0.0, group["betas"], group["eps"], group["weight_decay"])
        super().add_param_group(param_group)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed,
                "capturable": self.capturable, "last_norm": None}

    def _lr(self, group):
        """(learning rate as a number, as a tensor) of a group, one of them."""
        lr = group["lr"]
        if not isinstance(lr, Tensor):
            _check_hyper(lr, (0.0, 0.0), 0.0, 0.0)
            return lr, None
        if not self.capturable:
            raise ValueError("a learning rate in a tensor needs capturable=True")
        if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
            raise ValueError("a learning rate in a tensor is one float32 value on the GPU")
        return 0.0, lr

    def _state_of(self, p: Tensor, count: Optional[Tensor], capturing: bool) -> dict:
        state = self.state[p]
        if not state:
            if capturing:
                raise RuntimeError("step once before capturing a step: a capture would make the "
                                   "states anew at every replay")
            m, v = _STATES[self.state_bits]
            state["step"] = 0 if count is None else count
            state["exp_avg"] = torch.zeros_like(p, dtype=m, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=v, memory_format=torch.preserve_format)
            if self.state_bits == 8:
                blocks = (p.numel() + _BLOCK - 1) // _BLOCK
                for key in ("exp_avg_scale", "exp_avg_sq_scale"):
                    state[key] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return state

    def _count_of(self, group, device: torch.device) -> Tensor:
        """The group's count of steps on the GPU."""
        for p in group["params"]:
            if p in self.state:
                return self.state[p]["step"]
        return torch.zeros((), dtype=torch.int64, device=device)

    @torch.no_grad()
    def step(self, closure=None, *, max_norm: Optional[float] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_norm = None if max_norm is None else _check_max_norm(max_norm)
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("a captured step needs capturable=True: its count of steps would "
                               "stand still")
        call, params, stepped, numbers, groups, number = _Call(self.state_bits), [], [], [], [], 0
        for group in self.param_groups:
            lr, lr_device = self._lr(group)
            of = {}  # the call's group by count of steps
            count = None
            for p in group["params"]:
                number += 1
                if p.grad is None:
                    continue
                if self.capturable and count is None:
                    _on_one_gpu([p], "parameters")
                    if lr_device is not None and lr_device.device != p.device:
                        raise ValueError(f"a learning rate is on {lr_device.device}, its "
                                         f"parameters on {p.device}")
                    count = self._count_of(group, p.device)
                state = self._state_of(p, count, capturing)
                key = None if self.capturable else state["step"]
                if key not in of:
                    of[key] = call.group(
                        lr, group["betas"], group["eps"], group["weight_decay"],
                        0 if self.capturable else key + 1, lr_device, count)
                params.append(p)
                stepped.append(state)
                numbers.append(number - 1)
                groups.append(of[key])
        if not params:
            return loss
        grads = [p.grad for p in params]
        states = [[state[key] for state in stepped] for key in _KEYS[self.state_bits]]
        self.last_norm = grad_norm(grads) if max_norm is not None else None
        call.run(params, grads, states, numbers, groups, self.seed, self.last_norm,
                 max_norm or 0.0, self.capturable)
        if not self.capturable:
            for state in stepped:
                state["step"] += 1
        return loss

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # torch has cast the states to their parameters' types: take them as they were saved
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        m, v = _STATES[self.state_bits]
        for group in self.param_groups:
            count = None
            for p in group["params"]:
                was = state_dict["state"].get(saved.pop(0))
                if not was:
                    continue
                if was["exp_avg"].dtype != m or was["exp_avg_sq"].dtype != v:
                    raise ValueError(f"the saved states are {was['exp_avg'].dtype}: they need "
                                     f"another state_bits than {self.state_bits}")
                state = self.state[p]
                for key in ("exp_avg", "exp_avg_sq"):
                    if was[key].shape != p.shape:
                        raise ValueError(f"a saved {key} has shape {tuple(was[key].shape)}, its "
                                         f"parameter {tuple(p.shape)}")
                    state[key] = torch.empty_like(p, dtype=was[key].dtype,
                                                  memory_format=torch.preserve_format)
                    state[key].copy_(was[key])
                for key in ("exp_avg_scale", "exp_avg_sq_scale"):
                    if key in was:
                        state[key] = was[key].to(device=p.device, copy=True)
                step = int(was["step"])
                if self.capturable:
                    if count is None:
                        count = torch.full((), step, dtype=torch.int64, device=p.device)
                    elif step != int(count):
                        raise ValueError("capturable=True counts steps by group: the saved ones "
                                         "differ within one")
                    step = count
                state["step"] = step
