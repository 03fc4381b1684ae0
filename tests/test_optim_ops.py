"""What the steps over many tensors refuse, and what they check on the host: no GPU."""
import ctypes

import pytest
import torch

import tidegs_amd as tg
from tidegs_amd import _native as N

F8 = torch.float8_e4m3fn, torch.float8_e5m2


def _lists(n=10, dtype=torch.float32, state=torch.float32, device="cpu"):
    return ([torch.zeros(n, dtype=dtype, device=device)],
            [torch.zeros(n, dtype=dtype, device=device)],
            *([torch.zeros(n, dtype=state, device=device)] for _ in range(2)))


def _scales(blocks=1, **other):
    return dict(exp_avg_scales=[torch.zeros(blocks)], exp_avg_sq_scales=[torch.zeros(blocks)],
                **other)


def _eight(n=10):
    p, g, _, _ = _lists(n)
    return p, g, [torch.zeros(n).to(F8[0])], [torch.zeros(n).to(F8[1])]


@pytest.mark.parametrize("bad, match", [
    (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"), (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=-1.0), "weight_decay"), (dict(step=0), "steps count"),
    (dict(step=1 << 32), "steps count"), (dict(seed=-1), "seed"), (dict(seed=1 << 64), "seed"),
    (dict(max_norm=1.0), "go together"), (dict(grad_norm=torch.tensor(1.0)), "go together"),
    (dict(max_norm=0.0, grad_norm=torch.tensor(1.0)), "max_norm"),
    (dict(max_norm=float("nan"), grad_norm=torch.tensor(1.0)), "max_norm"),
    (dict(exp_avg_scales=[torch.zeros(1)]), "both states")])
def test_step_refuses_hyperparameters(bad, match):
    args = dict(step=1, lr=1e-3)
    args.update(bad)
    with pytest.raises(ValueError, match=match):
        tg.adamw_step(*_lists(), **args)


def test_step_refuses_tensors():
    p, g, m, v = _lists()
    with pytest.raises(ValueError, match="one length"):
        tg.adamw_step(p, g, m, [], 1, lr=1e-3)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.adamw_step(*_lists(dtype=torch.float64), 1, lr=1e-3)
    for grad in (torch.zeros(9), torch.zeros(10, dtype=torch.bfloat16),
                 torch.zeros(10, device="meta")):
        with pytest.raises(ValueError, match="gradient"):
            tg.adamw_step(p, [grad], m, v, 1, lr=1e-3)
    with pytest.raises(RuntimeError, match="sparse"):
        tg.adamw_step(p, [torch.zeros(10).to_sparse()], m, v, 1, lr=1e-3)
    for state in (torch.zeros(9), torch.zeros(10, dtype=torch.bfloat16),
                  torch.zeros(10, device="meta")):
        with pytest.raises(ValueError, match="exp_avg must"):
            tg.adamw_step(p, g, [state], v, 1, lr=1e-3)
        with pytest.raises(ValueError, match="exp_avg_sq must"):
            tg.adamw_step(p, g, m, [state], 1, lr=1e-3)
    with pytest.raises(ValueError, match="dense"):
        tg.adamw_step([torch.zeros(10, 2)[:, 0]], g, m, v, 1, lr=1e-3)
    with pytest.raises(ValueError, match="dense"):
        tg.adamw_step([torch.zeros(1).expand(10)], g, m, v, 1, lr=1e-3)
    with pytest.raises(ValueError, match="dense"):  # the state's order is another
        tg.adamw_step([torch.zeros(2, 5).t()], [torch.zeros(5, 2)], [torch.zeros(5, 2)],
                      [torch.zeros(5, 2)], 1, lr=1e-3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.adamw_step(p, g, m, v, 1, lr=1e-3)
    tg.adamw_step([], [], [], [], 1, lr=1e-3)  # nothing to do


def test_step_refuses_states_of_8_bits():
    p, g, m, v = _eight()
    with pytest.raises(ValueError, match="exp_avg must"):
        tg.adamw_step(p, g, v, v, 1, lr=1e-3, **_scales())
    with pytest.raises(ValueError, match="exp_avg_sq must"):
        tg.adamw_step(p, g, m, m, 1, lr=1e-3, **_scales())
    with pytest.raises(ValueError, match="exp_avg_scale must hold 1"):
        tg.adamw_step(p, g, m, v, 1, lr=1e-3, **_scales(2))
    with pytest.raises(ValueError, match="exp_avg_scale must hold 2"):
        tg.adamw_step(*_eight(129), 1, lr=1e-3, **_scales())
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.adamw_step(p, g, m, v, 1, lr=1e-3, **_scales())


def test_norm_refusals():
    with pytest.raises(ValueError, match="a tensor at least"):
        tg.grad_norm([])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.grad_norm([torch.zeros(3).int()])
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="one device"):
        tg.grad_norm([torch.zeros(3), torch.zeros(3, device="meta")])


def test_optimizer_refusals():
    p = torch.zeros(3, requires_grad=True)
    for bad, match in ((dict(lr=-1.0), "lr"), (dict(betas=(0.9, 1.0)), "betas"),
                       (dict(eps=-1.0), "eps"), (dict(weight_decay=-1.0), "weight_decay"),
                       (dict(state_bits=16), "state_bits"), (dict(seed=-1), "seed"),
                       (dict(lr=torch.tensor(1e-3)), "capturable"),
                       (dict(lr=torch.tensor(1e-3), capturable=True), "on the GPU")):
        with pytest.raises(ValueError, match=match):
            tg.AdamW([p], **bad)
    with pytest.raises(ValueError, match="betas"):
        tg.AdamW([dict(params=[p], betas=(0.9, 2.0))])
    opt = tg.AdamW([p])
    assert opt.step() is None  # no gradients: nothing to do
    assert opt.step(lambda: 3.0) == 3.0
    p.grad = torch.zeros(3)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    assert opt.state[p]["step"] == 0  # a refused step does not count


def test_optimizer_copies_and_loads():
    import copy
    import pickle

    p = torch.zeros(3, requires_grad=True)
    opt = tg.AdamW([p], state_bits=8, seed=5)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (other.state_bits, other.seed, other.capturable) == (8, 5, False)
        assert other.step() is None
    saved = dict(state={0: dict(step=1, exp_avg=torch.zeros(1), exp_avg_sq=torch.zeros(1))},
                 param_groups=tg.AdamW([p]).state_dict()["param_groups"])
    with pytest.raises(ValueError, match="shape"):
        tg.AdamW([p]).load_state_dict(saved)


def test_dense_orders():
    from tidegs_amd.optim_ops import _is_dense

    t = torch.zeros(4, 5, 6)
    for x in (t, t.permute(2, 0, 1), t[:1], t[:, :, :1][:1, :1], torch.zeros(0, 3), t[0].t(),
              torch.zeros(())):
        assert _is_dense(x)
    for x in (t[:, :3], t[..., ::2], torch.zeros(1).expand(4), t[:, 0]):
        assert not _is_dense(x)


def test_reader_of_lists():
    """What it does not read itself: the checks one by one follow."""
    from tidegs_amd.optim_ops import _lists

    r = _lists()
    t = [torch.zeros(3)]
    assert r.spans(t) is None and r.spans([]) is None and r.spans([3]) is None
    assert r.spans(t[0]) is None  # (rows of a tensor)
    assert r.adamw(t, t, t, t, None, None, 128, [0], [0]) is None
    assert r.adamw([], [], [], [], None, None, 128, [], []) is None
    with pytest.raises(TypeError):
        r.spans(3)
    with pytest.raises(TypeError, match="nine"):
        r.adamw(t, t)
    with pytest.raises(ValueError, match="one length"):
        r.adamw(t, t, t, [], None, None, 128, [0], [0])
    with pytest.raises(TypeError):
        r.adamw(t, t, t, t, None, None, "128", [0], [0])


def test_entry_points_check_their_arguments():
    lib = N.load()
    fake = 0x1000  # never dereferenced: the checks fail first

    class Tensor(ctypes.Structure):
        _fields_ = [(k, ctypes.c_void_p) for k in ("p", "g", "m", "v", "ms", "vs")] + [
            ("n", ctypes.c_uint64), ("number", ctypes.c_uint32), ("group", ctypes.c_uint32),
            ("dtype", ctypes.c_int32)]

    class Group(ctypes.Structure):
        _fields_ = [(k, ctypes.c_double) for k in ("lr", "b1", "b2", "eps", "wd")] + [
            ("step", ctypes.c_uint64), ("lr_device", ctypes.c_void_p),
            ("step_device", ctypes.c_void_p)]

    def step(bits=32, norm=None, max_norm=0.0, ws=None, ws_bytes=0, n_groups=1, group=(), **other):
        t = dict(p=fake, g=fake, m=fake, v=fake, ms=fake, vs=fake, n=5, number=0, group=0, dtype=0)
        t.update(other)
        h = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1)
        h.update(group)
        return lib.tgs_adamw(1, ctypes.byref(Tensor(**t)), n_groups, ctypes.byref(Group(**h)),
                             bits, 0, norm, max_norm, ws, ws_bytes, None)

    def refused(rc, text):
        assert rc < 0 and text in N.last_error(), N.last_error()

    refused(step(bits=16), "16 bits")
    refused(step(dtype=3), "dtype")
    refused(step(group=dict(step=0)), "step 0")
    refused(step(group=dict(step=1 << 32)), "step")
    refused(step(group=dict(b1=1.0)), "betas")
    refused(step(group=dict(eps=-1.0)), "eps")
    refused(step(group=dict(eps=float("nan"))), "eps")
    refused(step(group=dict(lr_device=fake)), "counted on the device")
    refused(step(group=dict(step_device=fake)), "workspace")
    refused(step(group=dict(step_device=fake), ws=fake + 8, ws_bytes=1 << 20), "16 bytes")
    refused(step(norm=fake), "max_norm")
    refused(step(n=1 << 42), "values")
    for name in ("p", "g", "m", "v"):
        refused(step(**{name: None}), "null")
    refused(step(bits=8, ms=None), "null")
    refused(step(bits=8, vs=None), "null")
    assert lib.tgs_adamw(0, None, 0, None, 32, 0, None, 0.0, None, 0, None) == 0
    assert step(n=0, p=None) == 0
    bad = Tensor(p=fake, g=fake, m=fake, v=fake, n=5, group=1)
    refused(lib.tgs_adamw(1, ctypes.byref(bad), 1, ctypes.byref(
        Group(lr=0.1, b1=0.9, b2=0.9, eps=0.1, step=1)), 32, 0, None, 0.0, None, 0, None),
        "group 1 of 1")

    class Span(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("n", ctypes.c_uint64), ("dtype", ctypes.c_int32)]

    need = lib.tgs_grad_norm_workspace_size(1)

    def norm(out=fake, ws=fake, ws_bytes=need, **other):
        s = dict(data=fake, n=5, dtype=0)
        s.update(other)
        return lib.tgs_grad_norm(1, ctypes.byref(Span(**s)), out, ws, ws_bytes, None)

    refused(norm(out=None), "null")
    refused(norm(data=None), "null")
    refused(norm(dtype=-1), "dtype")
    refused(norm(n=(1 << 38) + 1), "values")
    refused(norm(ws_bytes=need - 1), "workspace too small")
    refused(norm(ws=fake + 4), "8 bytes")
