"""What group norm refuses, and what it checks on the host: no GPU."""

import pytest
import torch

import tidegs_amd as tg
from tidegs_amd import _native as N


def test_refusals():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        tg.group_norm(x.double(), 2)
    with pytest.raises(ValueError, match="activation"):
        tg.group_norm(x, 2, activation="tanh")
    for bad in (torch.zeros(8), torch.tensor(1.0), torch.zeros(2, 5, 0), torch.zeros(1, 65537)):
        with pytest.raises(ValueError, match="channels"):
            tg.group_norm(bad, 1)
    for groups in (0, -1, 3, 16):
        with pytest.raises(ValueError, match="groups"):
            tg.group_norm(x, groups)
    for eps in (0.0, -1e-5, 1e-25, 1e25, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            tg.group_norm(x, 2, eps=eps)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tg.group_norm(x, 2)


def test_pixels_in_place_or_copied():
    """Which layouts are read where they lie, and at what distances."""
    from tidegs_amd.decoder_ops import _group_norm_node

    _pixels = _group_norm_node().pixels
    t = torch.arange(3 * 4 * 5 * 8.0).view(3, 4, 5, 8)
    for x, sample, pitch in (
            (t, 160, 8), (t[..., :6], 160, 8), (t[1:], 160, 8), (t[::2], 320, 8),
            (t[:, 1:3], 160, 8), (t[:, :, :1], 160, 40), (t[:, ::2], None, None),
            (t[:, :, 1:3], None, None), (t[:1].expand(3, 4, 5, 8), 0, 8), (t[:, 0, 0], 160, 8),
            (t[:, :1, :1, 2:5], 160, 3), (t.transpose(1, 2), None, None),
            (t[..., ::2], None, None), (t[..., :1].expand(3, 4, 5, 8), None, None),
            (t[:, :, :1].expand(3, 4, 5, 8), None, None)):
        y, s, p = _pixels(x)
        assert torch.equal(x, y)
        if sample is None:
            assert y.is_contiguous() and y.data_ptr() != x.data_ptr()
            assert (s, p) == (y.numel() // 3, y.shape[-1])
        else:
            assert y.data_ptr() == x.data_ptr()
            assert s == sample or x.shape[0] == 1
            assert p == pitch or x[0, ..., 0].numel() == 1
        # the values really are where the distances say
        flat = y.as_strided((y.untyped_storage().nbytes() // 4,), (1,), 0)
        pixels = x[0, ..., 0].numel()
        at = (y.storage_offset() + torch.arange(x.shape[0])[:, None, None] * s
              + torch.arange(pixels)[:, None] * p + torch.arange(x.shape[-1]))
        assert torch.equal(flat[at].reshape(x.shape), x)
    assert _pixels(torch.zeros(0, 3, 8))[1:] == (0, 8)


def test_node_checks_its_arguments():
    from tidegs_amd.decoder_ops import _group_norm_node

    node = _group_norm_node()
    with pytest.raises(TypeError, match="seven"):
        node.group_norm(torch.zeros(2, 4))
    with pytest.raises(TypeError, match="a tensor is needed"):
        node.group_norm(3, None, None, 1, 1e-5, 0, False)
    with pytest.raises(TypeError):
        node.group_norm(torch.zeros(2, 4), None, None, "1", 1e-5, 0, False)
    with pytest.raises(TypeError, match="six"):
        node.bind(1)


def test_entry_points_check_their_arguments():
    lib = N.load()
    fake = 0x1000  # never dereferenced: the checks fail first

    def refused(rc, text):
        assert rc < 0 and text in N.last_error(), N.last_error()

    def fwd(samples=2, pixels=4, width=8, groups=2, dtype=0, act=0, x=fake, pitch=8, wtype=None,
            eps=1e-5, y=fake, stats=None, ws=None, ws_bytes=0):
        return lib.tgs_group_norm_fwd(samples, pixels, width, groups, dtype, act, x, pixels * 8,
                                      pitch, None, None, dtype if wtype is None else wtype, eps,
                                      y, stats, ws, ws_bytes, None)

    def bwd(samples=2, pixels=4, width=8, groups=2, dtype=0, act=0, x=fake, pitch=8, dw=fake,
            dx=fake, stats=None, ws=fake, ws_bytes=1 << 40):
        return lib.tgs_group_norm_bwd(samples, pixels, width, groups, dtype, act, x, pixels * 8,
                                      pitch, fake, pixels * 8, pitch, None, None, dtype, 1e-5,
                                      stats, dx, dw, None, ws, ws_bytes, None)

    for call in (fwd, bwd):
        refused(call(dtype=3), "dtype")
        refused(call(dtype=-1), "dtype")
        refused(call(width=0), "width")
        refused(call(width=65544, groups=1), "width")
        refused(call(groups=0), "groups")
        refused(call(groups=3), "groups")
        refused(call(samples=1 << 40), "2^40")
        refused(call(act=4), "activation")
        refused(call(act=-1), "activation")
        refused(call(x=None), "null")
        refused(call(pitch=7), "pitch")
    refused(fwd(wtype=1), "weights")
    for eps in (0.0, 1e-30, 1e30, float("nan")):
        refused(fwd(eps=eps), "eps")
    refused(fwd(y=None), "null")
    assert fwd(samples=0, x=None, y=None) == 0 and fwd(pixels=0, x=None, y=None) == 0
    assert bwd(samples=0, dw=None) == 0 and bwd(dx=None, dw=None) == 0
    # groups too large for a team's registers
    large = dict(samples=2, pixels=10_000, width=8, groups=1)
    sizes = *large.values(), 0
    stats, need = lib.tgs_group_norm_stats_size(*sizes), lib.tgs_group_norm_fwd_workspace_size(
        *sizes)
    assert stats == 2 * 8 and need > 0
    refused(fwd(**large), "null stats")
    refused(fwd(**large, stats=fake, ws=fake, ws_bytes=need - 1), "workspace too small")
    refused(fwd(**large, stats=fake, ws=fake + 4, ws_bytes=need), "8 bytes")
    refused(fwd(**large, stats=fake + 4, ws=fake, ws_bytes=need), "8 bytes")
    need = lib.tgs_group_norm_bwd_workspace_size(*sizes)
    refused(bwd(**large, stats=fake, ws_bytes=need - 1), "workspace too small")
    refused(bwd(**large), "stats")
    refused(bwd(**large, stats=fake, ws=None), "8 bytes")
    # sizes that the calls refuse need nothing
    for bad in ((2, 4, 8, 3, 0), (2, 4, 8, 0, 0), (2, 4, 0, 1, 0), (2, 4, 8, 2, 5),
                (0, 4, 8, 2, 0), (2, 0, 8, 2, 0)):
        for query in ("stats_size", "fwd_workspace_size", "bwd_workspace_size"):
            assert getattr(lib, "tgs_group_norm_" + query)(*bad) == 0
    refused(lib.tgs_group_norm_bwd(2, 4, 8, 2, 0, 0, fake, 32, 8, fake, 32, 7, None, None, 0, 1e-5,
                                   None, fake, None, None, fake, 1 << 30, None), "pitch")
