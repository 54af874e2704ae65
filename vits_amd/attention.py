"""Attention with a learned relative position bias by buckets, forward and backward, on the HIP kernels
of csrc/bucket_attention_*.hip.

It stands next to the text encoder's windowed attention (``native.rel_attention``: learned key / value
embeddings within four positions, fp32, forward only): here the position enters as one learned number per
head and bucket of distances, any length is taken, key and value heads may be shared by groups of query
heads, and there is a backward pass.  Tensors are channel-major ``[batch, heads * head_dim, time]`` views
with dense time (slices of a fused projection go in as they are), fp32 or bf16.

    buckets = RelativeBuckets(32, 128)
    out = bucket_attention(q, k, v, bias, buckets, heads=8, key_lengths=n, query_lengths=n)

``bucket_attention`` records itself for autograd (reverse mode; forward-mode tangents are refused).  Recording
while a stream is captured into a HIP graph is refused: autograd's own accumulation nodes for leaves that an
earlier eager pass has touched would be captured with the stream of that pass.  A training step that is captured
calls ``bucket_attention`` under ``torch.no_grad()`` (with ``return_lse``) and ``bucket_attention_backward``.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import native


# Bucket tables by device and contents, a few KiB each, kept for good: a graph, or a call still running on another
# stream, may read one after the RelativeBuckets it was made for is gone.
_TABLES = {}


class RelativeBuckets:
    """Buckets of the offset key - query.  Half of the buckets are for keys ahead of the query, half for
    keys at or behind it (``bidirectional=False``: all for keys at or behind it, those ahead share bucket
    0).  Of a side's n buckets the first n // 2 hold one distance each, the others ranges whose borders grow
    in proportion up to ``max_distance``; everything further shares the last one.  The borders are found in
    whole numbers, so none depends on how a logarithm rounds."""

    def __init__(self, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True):
        side = num_buckets // 2 if bidirectional else num_buckets
        if num_buckets < (4 if bidirectional else 2) or (bidirectional and num_buckets % 2):
            raise ValueError("num_buckets must be at least 2 per direction, and even if bidirectional")
        if not side // 2 < max_distance <= native.BUCKET_MAX_DISTANCE:
            raise ValueError(f"max_distance must be above the single-distance buckets ({side // 2}) "
                             f"and at most {native.BUCKET_MAX_DISTANCE}")
        self.num_buckets, self.max_distance, self.bidirectional = num_buckets, max_distance, bidirectional
        single, ranges = side // 2, side - side // 2
        # distance n is in range r or further iff single * (max_distance / single) ** (r / ranges) <= n
        firsts, n = [], single
        for r in range(ranges):
            while n ** ranges * single ** r < max_distance ** r * single ** ranges:
                n += 1
            firsts.append(n)
        self._side = list(range(single))
        for n in range(single, max_distance + 1):
            self._side.append(single + sum(f <= n for f in firsts) - 1)
        self._tables = {}

    def bucket_of(self, offset: int) -> int:
        """The bucket of one offset key - query."""
        if offset > 0 and not self.bidirectional:
            return 0
        b = self._side[min(abs(offset), self.max_distance)]
        return b + self.num_buckets // 2 if offset > 0 else b

    def table(self, device) -> torch.Tensor:
        """int32 [2 * max_distance + 1] on ``device``: the bucket of every offset from -max_distance up.
        Made once per device, and there for good."""
        index = native._device_index(device)                # of "cuda" alone: the current device's, whichever that is
        t = self._tables.get(index)
        if t is None:
            # not even where another object has made this table: whether a call can be captured does not hang on that
            if torch.cuda.is_current_stream_capturing():
                raise native.NativeError("call RelativeBuckets.table(device) before the capture")
            of = tuple(self.bucket_of(o) for o in range(-self.max_distance, self.max_distance + 1))
            t = _TABLES.get((index, of))
            if t is None:
                with torch.inference_mode(False):           # a table first used there has to serve autograd too
                    t = _TABLES[index, of] = torch.tensor(of, dtype=torch.int32).to(torch.device("cuda", index))
            self._tables[index] = t
        return t


def _view3(name, t, dtype, device, shape=None):
    if t.dtype is dtype and t.device == device and t.dim() == 3 and (shape is None or t.shape == shape) \
            and (t.stride(2) == 1 or t.shape[2] <= 1):
        return
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be [batch, channels, time] of {dtype} on {device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must have a dense time axis, strides are {t.stride()}")


def _lengths(name, t, batch, device):
    if t is not None and (t.dtype != torch.int64 or t.device != device or tuple(t.shape) != (batch,) or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int64 tensor of {batch} on {device}")


def _check(q, k, v, bias, buckets, heads, kv_heads, key_lengths, query_lengths, query_start, scale):
    """Checks what both passes take; returns (kv_heads, scale, bucket table or None)."""
    if not q.is_cuda:
        raise native.NativeError("bucket_attention runs on the GPU only: there is no CPU fallback")
    dtype, device = q.dtype, q.device
    if dtype not in native.DTYPES:
        raise ValueError(f"q must be float32 or bfloat16, got {dtype}")
    kv_heads = heads if kv_heads is None else kv_heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    _view3("q", q, dtype, device)
    B, C, _ = q.shape
    if C % heads or not 1 <= C // heads <= native.BUCKET_MAX_HEAD_DIM:
        raise ValueError(f"q's {C} channels are not {heads} heads of 1..{native.BUCKET_MAX_HEAD_DIM}")
    _view3("k", k, dtype, device)
    shape = k.shape
    if shape[0] != B or shape[1] != C // heads * kv_heads:
        raise ValueError(f"k must be {(B, C // heads * kv_heads, shape[2])}, got {tuple(shape)}")
    _view3("v", v, dtype, device, shape)
    _lengths("key_lengths", key_lengths, B, device)
    _lengths("query_lengths", query_lengths, B, device)
    _lengths("query_start", query_start, B, device)
    table = None
    if (bias is None) != (buckets is None):
        raise ValueError("bias and buckets go together")
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.device != device or bias.shape != (heads, buckets.num_buckets) \
                or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous float32 [{heads}, {buckets.num_buckets}] on {device}")
        table = buckets.table(device)
    scale = (C // heads) ** -0.5 if scale is None else float(scale)
    if not 0 < scale < 1e30:
        raise ValueError("scale must be positive and finite")
    return kv_heads, scale, table


def _forward(q, k, v, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal, scale):
    out = native.empty_dense(q)
    lse = q.new_empty((q.shape[0], heads, q.shape[2]), dtype=torch.float32)
    native.bucket_attention(q, k, v, out, lse, bias, table, heads=heads, kv_heads=kv_heads, key_lengths=key_lengths,
                            query_lengths=query_lengths, query_start=query_start, causal=causal, scale=scale)
    return out, lse


def _backward(dout, q, k, v, out, lse, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal, scale):
    # gradients of sums come expanded, results of other code in another order
    dout, out = (t if t.stride(2) == 1 or t.shape[2] <= 1 else t.contiguous() for t in (dout, out))
    dq, dk, dv = native.empty_dense(q), native.empty_dense(k), native.empty_dense(v)
    dbias = torch.empty_like(bias) if bias is not None else None
    native.bucket_attention_backward(dout, q, k, v, out, lse, dq, dk, dv, bias, table, dbias, heads=heads, kv_heads=kv_heads,
                                     key_lengths=key_lengths, query_lengths=query_lengths, query_start=query_start,
                                     causal=causal, scale=scale)
    return dq, dk, dv, dbias


def _refuse_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise native.NativeError(f"{what} under autograd cannot be captured into a graph: call it under torch.no_grad() "
                                 "and its *_backward function")


def _refuse_forward_mode(what, *tensors):
    """Dual tensors of forward-mode differentiation do not say ``requires_grad``: without this, their tangents got lost."""
    if getattr(forward_ad, "_current_level", 0) >= 0 \
            and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise native.NativeError(f"{what} has no forward-mode derivative")


class _BucketAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal, scale):
        out, lse = _forward(q, k, v, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, bias, table, key_lengths, query_lengths, query_start)
        ctx.rest = heads, kv_heads, causal, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        _refuse_capture("the backward pass of bucket_attention")
        q, k, v, out, lse, bias, table, key_lengths, query_lengths, query_start = ctx.saved_tensors
        heads, kv_heads, causal, scale = ctx.rest
        dq, dk, dv, dbias = _backward(dout, q, k, v, out, lse, bias, table, heads, kv_heads, key_lengths, query_lengths,
                                      query_start, causal, scale)
        return dq, dk, dv, dbias, None, None, None, None, None, None, None, None


def bucket_attention(q, k, v, bias=None, buckets: RelativeBuckets | None = None, *, heads: int, kv_heads: int | None = None,
                     key_lengths=None, query_lengths=None, query_start=None, causal: bool = False,
                     scale: float | None = None, return_lse: bool = False):
    """Attention of q ``[B, heads * D, Tq]`` over k, v ``[B, kv_heads * D, Tk]``: the logit of query i and key j is
    ``scale * q_i . k_j + bias[head, buckets.bucket_of(j - pos_i)]`` with ``pos_i = query_start[b] + i`` (0 + i without
    it), over j < key_lengths[b] and, with ``causal``, j <= pos_i.

    bias: float32 ``[heads, buckets.num_buckets]``, or None (no position bias); -inf or a type's lowest value (below -2.36e38)
    forbids a bucket, and a query that may see nothing else is one without a key.  key_lengths, query_lengths, query_start:
    int64 ``[B]`` on the device, or None.  scale: 1 / sqrt(D) unless given, positive.  Queries without a key and those at or behind
    query_lengths[b] come out as zero.  What lies behind a length enters no result, nor do keys that ``causal`` hides from all
    of an item's queries: padding may hold anything.  Serving a new token over a cache: Tq = 1, query_start = key_lengths - 1;
    the cache may be a view of a larger buffer.

    Returns out ``[B, heads * D, Tq]``, with ``return_lse`` also the log-sum-exp of the logits ``[B, heads, Tq]`` (-inf
    where there is no key), which ``bucket_attention_backward`` takes and which carries no gradient."""
    kv_heads, scale, table = _check(q, k, v, bias, buckets, heads, kv_heads, key_lengths, query_lengths, query_start, scale)
    _refuse_forward_mode("bucket_attention", q, k, v, bias)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        _refuse_capture("bucket_attention")
        out, lse = _BucketAttention.apply(q, k, v, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start,
                                          causal, scale)
    else:
        out, lse = _forward(q, k, v, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal, scale)
    return (out, lse) if return_lse else out


def bucket_attention_backward(dout, q, k, v, out, lse, bias=None, buckets: RelativeBuckets | None = None, *, heads: int,
                              kv_heads: int | None = None, key_lengths=None, query_lengths=None, query_start=None,
                              causal: bool = False, scale: float | None = None):
    """Gradients (dq, dk, dv, dbias) of ``bucket_attention`` for the gradient ``dout`` of its output, from what it took
    and gave (``out``, ``lse``); dbias is None without a bias.  dout and out may have any strides (without a dense time
    axis they are copied).  Every sum has a fixed order: the same inputs give the
    same bits.  Padding gets zero gradients, and so does a query all of whose keys have a bias so low that lse < -2^20: fp32
    does not hold its probabilities there."""
    kv_heads, scale, table = _check(q, k, v, bias, buckets, heads, kv_heads, key_lengths, query_lengths, query_start, scale)
    _refuse_forward_mode("bucket_attention_backward", dout, q, k, v, out, lse, bias)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must be {tuple(q.shape)} of {q.dtype} on {q.device}")
    if tuple(lse.shape) != (q.shape[0], heads, q.shape[2]) or lse.dtype != torch.float32 or not lse.is_contiguous() \
            or lse.device != q.device:
        raise ValueError(f"lse must be a contiguous float32 [{q.shape[0]}, {heads}, {q.shape[2]}] on {q.device}")
    return _backward(dout, q, k, v, out, lse, bias, table, heads, kv_heads, key_lengths, query_lengths, query_start, causal,
                     scale)
