"""The norms around a transformer block, its gate, residual scale and residual sum, as one operator with a
backward pass, on the HIP kernels of csrc/block_norm.hip.

    z = norm(y) * post_weight + post_bias     y: what the block put out
    h = x + scale * gate * z                  x: the residual stream
    n = norm(h) * pre_weight + pre_bias       what the next block reads

It stands next to ``native.channel_norm`` (LayerNorm over 192 channels, fp32, forward only).  Tensors are channel-major
``[batch, channels, time]`` views with dense time, fp32 or bf16; the norms run over the channels.

``block_norm`` records itself for autograd (reverse mode; forward-mode tangents are refused); recording while a stream
is captured into a HIP graph is refused (see ``vits_amd.attention``): capture ``block_norm`` under ``torch.no_grad()`` and
``block_norm_backward``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import native
from .attention import _lengths, _refuse_capture, _refuse_forward_mode, _view3

_NORMS = {"layer": native.NORM_LAYER, "rms": native.NORM_RMS}


class BlockNormGrads(NamedTuple):
    """Gradients of ``block_norm``; None for what was not given."""
    x: torch.Tensor
    y: torch.Tensor | None
    gate: torch.Tensor | None
    scale: torch.Tensor | None
    post: tuple | None              # (weight, bias or None)
    pre: tuple | None


def _dense(t):
    return t if t is None or t.shape[2] <= 1 or t.stride(2) == 1 else t.contiguous()


def _param(name, t, channels, device):
    if t is not None and (t.dtype is not torch.float32 or t.device != device or t.shape != (channels,) or not t.is_contiguous()):
        raise ValueError(f"{name} (or its weight or bias) must be a contiguous float32 [{channels}] on {device}")


def _check(like, y, gate, scale, post, pre, norm, eps, lengths):
    if not like.is_cuda:
        raise native.NativeError("block_norm runs on the GPU only: there is no CPU fallback")
    if like.dtype not in native.DTYPES:
        raise ValueError(f"x must be float32 or bfloat16, got {like.dtype}")
    dtype, device = like.dtype, like.device
    _view3("x", like, dtype, device)
    shape = like.shape
    B, C, T = shape
    if not 1 <= C <= native.BLOCK_NORM_MAX_CHANNELS:
        raise ValueError(f"channels must be 1..{native.BLOCK_NORM_MAX_CHANNELS}, got {C}")
    if y is None:
        if gate is not None or scale is not None or post is not None:
            raise ValueError("gate, scale and post go with y")
    else:
        _view3("y", y, dtype, device, shape)
    if gate is not None:
        _view3("gate", gate, dtype, device)
        if gate.shape != shape and gate.shape != (B, C, 1):
            raise ValueError(f"gate must be {(B, C, T)} or {(B, C, 1)}, got {tuple(gate.shape)}")
    _param("scale", scale, C, device)
    for name, pair in (("post", post), ("pre", pre)):
        if pair is not None:
            if pair[0] is None:
                raise ValueError(f"{name} is (weight, bias or None)")
            _param(name, pair[0], C, device)
            _param(name, pair[1], C, device)
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)}")
    if not 0 < eps < 1e30:
        raise ValueError("eps must be positive and finite")
    if y is None and pre is None:
        raise ValueError("nothing to do: neither y nor pre is given")
    _lengths("lengths", lengths, B, device)


def _forward(x, y, gate, scale, post, pre, norm, eps, lengths):
    h = native.empty_dense(x) if y is not None else None
    n = native.empty_dense(x) if pre is not None else None
    native.block_norm(x, y, h, n, gate=gate, scale=scale, post=post, pre=pre, norm=_NORMS[norm], eps=eps, lengths=lengths)
    return h, n


def _backward(dh, dn, h, y, gate, scale, post, pre, norm, eps, lengths):
    dh, dn = _dense(dh), _dense(dn)
    like = dh if dh is not None else dn
    new = lambda t: native.empty_dense(t) if t is not None else None  # noqa: E731
    dx, dy, dgate = new(like), new(y), new(gate)
    row = iter(like.new_empty((5, like.shape[1]), dtype=torch.float32).unbind(0))     # the parameters' gradients: one allocation
    par = lambda t: next(row) if t is not None else None  # noqa: E731
    dscale = par(scale)
    dpost = (par(post[0]), par(post[1])) if post is not None else None
    dpre = (par(pre[0]), par(pre[1])) if pre is not None and dn is not None else None
    native.block_norm_backward(dh, dn, h, y, dx, dy, gate=gate, dgate=dgate, scale=scale, dscale=dscale, post=post, dpost=dpost,
                               pre=pre if dn is not None else None, dpre=dpre, norm=_NORMS[norm], eps=eps, lengths=lengths)
    return BlockNormGrads(dx, dy, dgate, dscale, dpost, dpre)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, w_post, b_post, w_pre, b_pre, norm, eps, lengths):
        ctx.set_materialize_grads(False)
        post = (w_post, b_post) if w_post is not None else None
        pre = (w_pre, b_pre) if w_pre is not None else None
        h, n = _forward(x, y, gate, scale, post, pre, norm, eps, lengths)
        ctx.save_for_backward(x if h is None else h, y, gate, scale, w_post, b_post, w_pre, b_pre, lengths)
        ctx.rest = norm, eps
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        _refuse_capture("the backward pass of block_norm")
        if dh is None and dn is None:
            return (None,) * 11
        h, y, gate, scale, w_post, b_post, w_pre, b_pre, lengths = ctx.saved_tensors
        norm, eps = ctx.rest
        post = (w_post, b_post) if w_post is not None else None
        pre = (w_pre, b_pre) if w_pre is not None else None
        g = _backward(dh, dn, h, y, gate, scale, post, pre, norm, eps, lengths)
        dpost, dpre = g.post or (None, None), g.pre or (None, None)
        return g.x, g.y, g.gate, g.scale, *dpost, *dpre, None, None, None


def block_norm(x, y=None, *, post=None, gate=None, scale=None, pre=None, norm: str = "layer", eps: float = 1e-5, lengths=None):
    """(h, n): h = x + scale * gate * norm(y), n = norm(h), see above.

    x, y: ``[B, C, T]``.  post, pre: (weight, bias) of the norm after the block and of the one before the next, bias may be
    None; without ``post`` y is taken as it is, without ``pre`` n is None.  gate: ``[B, C, T]`` or ``[B, C, 1]`` (one value per
    item and channel); scale: ``[C]``.  Parameters are float32.  Without y there is only the norm of x: h is x itself.
    norm: "layer" or "rms".  Columns at or behind ``lengths[b]`` (int64 ``[B]``) enter no result and come out as
    zero; padding, and the gate of an item without columns, may hold anything."""
    _check(x, y, gate, scale, post, pre, norm, eps, lengths)
    w_post, b_post = post or (None, None)
    w_pre, b_pre = pre or (None, None)
    _refuse_forward_mode("block_norm", x, y, gate, scale, w_post, b_post, w_pre, b_pre)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, y, gate, scale, w_post, b_post, w_pre, b_pre)):
        _refuse_capture("block_norm")
        h, n = _BlockNorm.apply(x, y, gate, scale, w_post, b_post, w_pre, b_pre, norm, eps, lengths)
    else:
        h, n = _forward(x, y, gate, scale, post, pre, norm, eps, lengths)
    return (x if h is None else h), n


def block_norm_backward(dh, dn, h, y=None, *, post=None, gate=None, scale=None, pre=None, norm: str = "layer", eps: float = 1e-5,
                        lengths=None) -> BlockNormGrads:
    """Gradients of ``block_norm`` for the gradients dh, dn of its outputs (either may be None), from the h it gave (x where
    there was no y) and what it took.  Sums over columns have a fixed order: the same inputs give the same bits.  Without
    dn there is no gradient of ``pre``.  With a gate ``[B, C, 1]`` and T > 1, B is at most 65530."""
    if dh is None and dn is None:
        raise ValueError("no gradient came in")
    if dn is not None and pre is None:
        raise ValueError("dn needs pre")
    _check(h, y, gate, scale, post, pre, norm, eps, lengths)
    _refuse_forward_mode("block_norm_backward", dh, dn, h, y, gate, scale, *(post or ()), *(pre or ()))
    for name, t in (("dh", dh), ("dn", dn)):
        if t is not None and (tuple(t.shape) != tuple(h.shape) or t.dtype != h.dtype or t.device != h.device):
            raise ValueError(f"{name} must be {tuple(h.shape)} of {h.dtype} on {h.device}")
    return _backward(dh, dn, h, y, gate, scale, post, pre, norm, eps, lengths)
