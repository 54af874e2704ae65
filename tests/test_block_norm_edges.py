"""The norms around a block at the edges of their definition.  The 64-bit reference and the derived bounds are those of
test_block_norm.py."""
import ctypes as C
import math

import pytest
import torch

from test_block_norm import _args, assert_within, grads_dict, inputs, reference
from vits_amd import native
from vits_amd.block_norm import block_norm, block_norm_backward

gpu = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@gpu
@TYPES
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("val", [math.nan, math.inf])
def test_the_gate_of_an_empty_item_may_hold_anything(val, norm, dtype):
    """A gate per item that was, say, a mean over no columns: it is not part of any sum."""
    lengths = torch.tensor([37, 0, 21], device="cuda")
    d, dh, dn = inputs(dtype, 3, 96, 37, gate="item")
    h, n = block_norm(**d, norm=norm, lengths=lengths)
    keep = {k: v for k, v in d.items() if k not in ("x", "y")}
    want = grads_dict(block_norm_backward(dh, dn, h, d["y"], **keep, norm=norm, lengths=lengths))
    ref = reference(None, d["y"], d["gate"], d["scale"], d["post"], d["pre"], norm, 1e-5, lengths, dh, dn, h)
    d["gate"] = d["gate"].clone()
    d["gate"][1] = val
    keep["gate"] = d["gate"]
    h2, n2 = block_norm(**d, norm=norm, lengths=lengths)
    assert torch.equal(h2, h) and torch.equal(n2, n)
    got = grads_dict(block_norm_backward(dh, dn, h, d["y"], **keep, norm=norm, lengths=lengths))
    for name in want:
        assert_within(name, got[name], ref[name])
        assert torch.equal(got[name], want[name]), name


@gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    d, dh, dn = inputs(torch.float32, 1, 16, 8)
    h, n = block_norm(**d)
    keep = {k: v for k, v in d.items() if k not in ("x", "y")}
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for name in ("x", "y", "gate", "scale"):
            with pytest.raises(native.NativeError, match="forward"):
                block_norm(**(d | {name: dual(d[name])}))
        for name in ("post", "pre"):
            for i in range(2):
                pair = list(d[name])
                pair[i] = dual(pair[i])
                with pytest.raises(native.NativeError, match="forward"):
                    block_norm(**(d | {name: tuple(pair)}))
        for args in ((dual(dh), dn, h, d["y"]), (dh, dual(dn), h, d["y"]), (dh, dn, dual(h), d["y"]), (dh, dn, h, dual(d["y"]))):
            with pytest.raises(native.NativeError, match="forward"):
                block_norm_backward(*args, **keep)
        assert torch.equal(block_norm(**d)[0], h)


def test_c_entries_refuse_negative_and_endless_strides():
    L = native.lib()
    room = dict(workspace=4096, workspace_bytes=1 << 40)
    F = lambda **kw: L.vk_block_norm(C.byref(_args(**kw)), None)
    B = lambda **kw: L.vk_block_norm_backward(C.byref(_args(**kw, **room)), None)
    for n in ("x", "y", "gate", "h", "n"):
        assert F(**{n + "_cstride": -100}) == -1 and F(**{n + "_bstride": -6400}) == -1, n
        assert F(**{n + "_cstride": 1 << 61}) == -1, n
    for n in ("y", "gate", "h", "dh", "dn", "dx", "dy", "dgate"):
        assert B(**{n + "_cstride": -100}) == -1 and B(**{n + "_bstride": -6400}) == -1, n
        assert B(**{n + "_cstride": 1 << 61}) == -1, n


def test_the_workspace_query_refuses_what_the_pass_refuses():
    L = native.lib()
    for bad, code in ((dict(length=(1 << 31) - 1), -2), (dict(length=(1 << 28) + 1), -2), (dict(dtype=7), -2), (dict(channels=4097), -2),
                      (dict(batch=-1), -1)):
        a = _args(**bad)
        assert L.vk_block_norm_backward_workspace_bytes(C.byref(a)) == code, bad
        assert L.vk_block_norm_backward(C.byref(a), None) == code, bad
