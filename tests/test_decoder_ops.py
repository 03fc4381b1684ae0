"""What the decoder operators refuse, and what they check on the host: no GPU."""
import ctypes

import pytest
import torch

import tidegs_amd as tg
from tidegs_amd import _native as N


def _ffn(width=8, hidden=16, out=3, dtype=torch.float32, **other):
    t = dict(x=torch.zeros(4, width, dtype=dtype), w_gate=torch.zeros(hidden, width, dtype=dtype),
             w_up=torch.zeros(hidden, width, dtype=dtype),
             w_down=torch.zeros(out, hidden, dtype=dtype))
    t.update(other)
    return t


def test_layer_norm_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.layer_norm(x.double())
    with pytest.raises(ValueError, match="last dimension"):
        tg.layer_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="last dimension"):
        tg.layer_norm(torch.tensor(1.0))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            tg.layer_norm(x, eps=eps)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.layer_norm(x)


def test_dropout_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.dropout(x.int(), 0.1, 1)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match=r"\[0, 1\]"):
            tg.dropout(x, p, 1)
    for seed, offset in ((-1, 0), (1 << 64, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError, match="64-bit"):
            tg.dropout(x, 0.1, seed, offset)
    for residual in (torch.zeros(8, 4), torch.zeros(4, 8, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="residual"):
            tg.dropout(x, 0.1, 1, residual=residual)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.dropout(x, 0.1, 1)


def test_gated_ffn_refusals():
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.gated_ffn(**_ffn(dtype=torch.float64))
    with pytest.raises(ValueError, match="activation"):
        tg.gated_ffn(**_ffn(), activation="tanh")
    for bad in (dict(width=0), dict(hidden=0), dict(out=0), dict(hidden=70000)):
        with pytest.raises(ValueError, match="must lie in"):
            tg.gated_ffn(**_ffn(**bad))
    with pytest.raises(ValueError, match="the weights two"):
        tg.gated_ffn(**_ffn(w_down=torch.zeros(16)))
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.gated_ffn(**_ffn())


def test_parameters_are_checked():
    """Shape, type and device of a weight, as the operators check them."""
    from tidegs_amd.decoder_ops import _parameter

    x = torch.zeros(4, 8)
    assert _parameter(None, "w", (8,), x) is None
    assert _parameter(torch.zeros(8, 16)[:, ::2], "w", (8, 8), x).is_contiguous()
    with pytest.raises(ValueError, match="w must have shape"):
        _parameter(torch.zeros(7), "w", (8,), x)
    with pytest.raises(TypeError, match="w must be torch.float32"):
        _parameter(torch.zeros(8, dtype=torch.bfloat16), "w", (8,), x)
    with pytest.raises(ValueError, match="w is on"):
        _parameter(torch.zeros(8, device="meta"), "w", (8,), x)
    _parameter(torch.zeros(8), "w", (8,), x.bfloat16(), (torch.float32,))


def test_rows_in_place_or_copied():
    """Which layouts are read where they lie."""
    from tidegs_amd.decoder_ops import _rows

    t = torch.arange(24 * 64.0).view(24, 64)
    view, rows, pitch = _rows(t[:, :59])
    assert view.data_ptr() == t.data_ptr() and (rows, pitch) == (24, 64)
    same, rows, pitch = _rows(t.view(2, 12, 64))
    assert same.data_ptr() == t.data_ptr() and (rows, pitch) == (24, 64)
    for other in (t.t(), t[:, ::2], t[:1].expand(5, 64), t.view(2, 12, 64)[:, :, :59]):
        copy, rows, pitch = _rows(other)
        assert copy.data_ptr() != t.data_ptr() and torch.equal(copy, other)
        assert (rows, pitch) == (other.numel() // other.shape[-1], other.shape[-1])
    assert _rows(torch.zeros(0, 8))[1:] == (0, 8)
    assert _rows(torch.zeros(3, 0))[1] == 0


def test_entry_points_check_their_arguments():
    lib = N.load()
    fake = ctypes.c_void_p(0x1000)  # never dereferenced: the checks fail first

    def refused(rc, text):
        assert rc < 0 and text in N.last_error(), N.last_error()

    def norm(rows=4, width=8, dtype=0, x=fake, pitch=8, wtype=0, y=fake):
        return lib.tgs_layer_norm_fwd(rows, width, dtype, x, pitch, None, None, wtype, 1e-5, y,
                                      None)

    refused(norm(dtype=3), "dtype")
    refused(norm(width=0), "width")
    refused(norm(wtype=1), "weights")
    refused(norm(x=None), "null")
    refused(norm(pitch=7), "pitch")
    assert norm(rows=0, x=None, y=None) == 0
    need = lib.tgs_layer_norm_bwd_workspace_size(4, 8)
    refused(lib.tgs_layer_norm_bwd(4, 8, 0, fake, 8, fake, 8, None, 0, 1e-5, None, fake, None,
                                   fake, need - 1, None), "workspace too small")
    assert lib.tgs_layer_norm_bwd(0, 8, 0, None, 8, None, 8, None, 0, 1e-5, fake, None, None,
                                  None, 0, None) == 0

    refused(lib.tgs_dropout(8, 5, fake, None, fake, 1, 0, 0, None), "dtype")
    refused(lib.tgs_dropout(8, 0, fake, None, fake, 65537, 0, 0, None), "threshold")
    refused(lib.tgs_dropout(8, 0, None, None, fake, 1, 0, 0, None), "null")
    assert lib.tgs_dropout(0, 0, None, None, None, 1, 0, 0, None) == 0

    def ffn(rows=4, width=8, hidden=16, out=3, dtype=0, act=0, x=fake, pitch=8, ws=1 << 30):
        return lib.tgs_gated_ffn_fwd(rows, width, hidden, out, dtype, act, x, pitch, fake, fake,
                                     fake, None, None, None, fake, fake, ws, None)

    refused(ffn(dtype=-1), "dtype")
    refused(ffn(act=3), "activation")
    refused(ffn(hidden=0), "positive")
    refused(ffn(width=65537), "65536")
    refused(ffn(rows=1 << 31), "rows")
    refused(ffn(x=None), "null")
    refused(ffn(pitch=7), "pitch")
    if lib.tgs_gated_ffn_fwd_workspace_size(4, 8, 16, 3, 0):
        refused(ffn(ws=0), "workspace too small")
    assert ffn(rows=0) == 0
    refused(lib.tgs_gated_ffn_fwd(4, 8, 16, 3, 0, 0, fake, 8, fake, fake, fake, None, None, None,
                                  fake, ctypes.c_void_p(0x1008), 1 << 30, None), "16 bytes")


def test_workspace_sizes_never_shrink_with_the_rows():
    lib = N.load()
    rows = sorted({max(1, (1 << k) + d) for k in range(24) for d in (-1, 0, 1)})
    for width in (1, 59, 64, 1000, 5000):
        got = [lib.tgs_layer_norm_bwd_workspace_size(r, width) for r in rows]
        assert got == sorted(got)
    for sizes in ((59, 128, 3), (64, 256, 48), (1024, 4096, 1024), (7, 33, 5)):
        for dtype in (0, 1, 2):
            for query in (lib.tgs_gated_ffn_fwd_workspace_size,
                          lib.tgs_gated_ffn_bwd_workspace_size):
                got = [query(r, *sizes, dtype) for r in rows]
                assert got == sorted(got), (sizes, dtype)


def test_tangents_are_refused_not_lost(monkeypatch):
    """Forward-mode differentiation raises, whichever input carries the tangent and whether
    or not a gradient is asked for as well; calls without tangents pass inside a level.  The
    launches are left out."""
    from torch.autograd import forward_ad

    from tidegs_amd import decoder_ops

    monkeypatch.setattr(decoder_ops, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(N, "call", lambda *a: 0)
    monkeypatch.setattr(N, "stream_handle", lambda *a: 0)
    x, w, b = torch.randn(4, 8), torch.ones(8), torch.zeros(8)
    ffn = list(_ffn().values()) + [torch.zeros(n) for n in (16, 16, 3)]
    calls = [(tg.layer_norm, [x, w, b]),
             (lambda x, r: tg.dropout(x, 0.1, 1, residual=r), [x, torch.randn(4, 8)]),
             (tg.gated_ffn, ffn)]
    for op, tensors in calls:
        for i, t in enumerate(tensors):
            for mode in (torch.enable_grad, torch.no_grad):
                for needs in (False, True):
                    with mode(), forward_ad.dual_level():
                        op(*tensors)
                        moved = list(tensors)
                        moved[i] = forward_ad.make_dual(t.clone().requires_grad_(needs),
                                                        torch.ones_like(t))
                        with pytest.raises(NotImplementedError, match="jvp"):
                            op(*moved)
        with torch.no_grad():
            assert not op(*tensors).requires_grad


def test_workspace_sizes_of_refused_sizes():
    """Nothing for what the calls refuse, with the reason (a hidden size of 0 ended the process)."""
    lib = N.load()
    for query in (lib.tgs_gated_ffn_fwd_workspace_size, lib.tgs_gated_ffn_bwd_workspace_size):
        for rows, width, hidden, out, dtype, text in (
                (4, 64, 0, 64, 1, "positive"), (4, 0, 0, 0, 0, "positive"), (4, 200, 16, 0, 0, "positive"),
                (4, 65537, 16, 3, 0, "65536"), (4, 1 << 31, 1 << 31, 1 << 31, 2, "65536"),
                (1 << 31, 64, 64, 64, 0, "rows"), (1 << 63, 64, 64, 64, 0, "rows"),
                (4, 64, 64, 64, 7, "dtype")):
            assert query(rows, width, hidden, out, dtype) == 0 and text in N.last_error()
        for dtype in (0, 1, 2):
            assert query(0, 64, 64, 64, dtype) > 0 and query(4, 65536, 65536, 65536, dtype) > 0


def test_six_products_of_planes_keep_24_bits():
    """The arithmetic of float32 products, on the host: three bfloat16 planes, each what the
    ones before leave, rounded, are the value; the products left out come to 2^-24 at most."""
    g = torch.Generator().manual_seed(1)
    for spread in (2.0 ** -8, 2.0 ** -7, 1.0):  # the worst lie just below 1 + 2^-8
        planes = []
        for _ in range(2):
            v = 1 + spread * torch.rand(1 << 20, generator=g)
            rest, parts = v.clone(), []
            for _ in range(3):
                parts.append(rest.to(torch.bfloat16).float())
                rest = rest - parts[-1]
            assert not bool(rest.any())
            planes.append([p.double() for p in parts])
        a, b = planes
        kept = a[0] * b[2] + a[2] * b[0] + a[1] * b[1] + a[1] * b[0] + a[0] * b[1] + a[0] * b[0]
        want = sum(a) * sum(b)
        assert float(((kept - want) / want).abs().max()) <= 2.0 ** -24
