"""Bucketed-bias attention at the edges of its definition.  The 64-bit reference and the derived bounds are those of
test_bucket_attention.py."""
import ctypes as C
import math

import pytest
import torch

from test_bucket_attention import _args, assert_within, both, i64, inputs, ref_of
from vits_amd import attention, native
from vits_amd.attention import RelativeBuckets, bucket_attention, bucket_attention_backward

gpu = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
GRADS = ("dq", "dk", "dv", "dbias")


# ---- keys that end just outside the table's reach, in a tile that goes on into it -------------------

@gpu
@TYPES
@pytest.mark.parametrize("Tq", [1, 5])
@pytest.mark.parametrize("nk", [300, 301, 999])
def test_keys_far_behind_the_queries(nk, Tq, dtype):
    """Positions around nk + max_distance: the last keys are at the last bucket's border, and the tile that holds them
    reaches back into the table."""
    far, span = 128, 128 if dtype == torch.bfloat16 else 64                 # positions of a tile
    starts = list(range(nk + far - 4, nk + far + span + 2, 7))
    case = (len(starts), 2, 1, 64, Tq, nk + 3, (32, far, True), False, [nk] * len(starts), None, starts)
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    assert_within("lse", lse, ref["lse"])
    assert_within("out", out, ref["out"])
    for name, g in zip(GRADS, bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)):
        assert_within(name, g, ref[name])


@gpu
@TYPES
@pytest.mark.parametrize("nk", [100, 33])
def test_more_queries_than_keys(nk, dtype):
    """A short memory: rows far behind the last key, without query_start and without query_lengths."""
    case = (1, 2, 2, 64, 300, 300, (32, 128, True), False, [nk], None, None)
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    assert_within("lse", lse, ref["lse"])
    assert_within("out", out, ref["out"])


# ---- biases that forbid ----------------------------------------------------------------------------

FORBID = [-math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min]
# B, H, Hk, D, Tq, Tk, buckets, causal, nk, nq, start: rows behind nk + max_distance see only the last bucket of the keys behind
FORBID_CASES = [
    (1, 2, 1, 64, 300, 300, (16, 40, True), False, [150], None, None),
    (2, 2, 2, 96, 131, 131, (8, 20, True), False, [90, 131], None, None),
    (1, 4, 2, 128, 200, 200, (16, 40, True), True, [130], None, None),
    (9, 16, 4, 128, 257, 257, (16, 40, True), True, None, None, None),
    (17, 16, 8, 64, 130, 130, (16, 40, True), False, None, None, None),
]
FORBID_IDS = [f"B{c[0]}H{c[1]}-{c[2]}D{c[3]}T{c[4]}{'c' if c[7] else ''}" for c in FORBID_CASES]


@gpu
@TYPES
@pytest.mark.parametrize("value", FORBID, ids=["inf", "lowest32", "lowest16"])
@pytest.mark.parametrize("which", ["behind", "ahead", "both"])
@pytest.mark.parametrize("case", FORBID_CASES, ids=FORBID_IDS)
def test_a_forbidden_bucket(case, which, value, dtype):
    """The bucket of everything far behind, of everything far ahead, or both, at -inf or at a type's lowest value.
    A row of which nothing is left is a row without keys.

    The reference takes -800 for the forbidden value: next to any other key of a row the probability is 0 in 64 bits too
    (logits here are below 30 in magnitude), and the rows that have no other key are behind the reference's query_lengths."""
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    side, far, B, Tq = buckets.num_buckets // 2, buckets.max_distance, case[0], case[4]
    gone = [b for b, at in ((side - 1, "behind"), (2 * side - 1, "ahead")) if which in (at, "both")]
    finite = bias.clone()
    finite[:, gone] = -800.0
    bias[:, gone] = value
    first = buckets._side.index(side - 1)                   # the distance at which the last bucket begins
    nk = case[8] or [case[5]] * B
    ref_opts = opts | dict(query_lengths=i64([min(Tq, n - 1 + first) if which != "ahead" else Tq for n in nk]))
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, finite, buckets, ref_opts, dout)
    assert_within("lse", lse, ref["lse"])
    assert_within("out", out, ref["out"])
    grads = dict(zip(GRADS, bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)))
    for name in GRADS:
        assert_within(name, grads[name], ref[name])
    assert not grads["dbias"][:, gone].any()


@gpu
@TYPES
@pytest.mark.parametrize("value", FORBID, ids=["inf", "lowest32", "lowest16"])
def test_everything_forbidden(value, dtype):
    """One head's whole bias forbids: its rows are without keys; the other head is as it was."""
    for case in ((1, 2, 2, 64, 70, 70, (16, 40, True), False, None, None, None),
                 (2, 2, 2, 128, 1, 1000, (16, 40, False), True, None, None, [999, 500]),
                 (9, 16, 16, 128, 257, 257, (16, 40, True), False, None, None, None)):
        q, k, v, bias, dout, buckets, opts = both(case, dtype)
        D = case[3]
        want, want_lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
        want_grads = bucket_attention_backward(dout, q, k, v, want, want_lse, bias, buckets, **opts)
        bias[0] = value
        out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
        assert not out[:, :D].any() and (lse[:, 0] == -math.inf).all()
        assert torch.equal(out[:, D:], want[:, D:]) and torch.equal(lse[:, 1:], want_lse[:, 1:])
        dq, dk, dv, dbias = bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)
        assert not dq[:, :D].any() and not dbias[0].any()
        assert torch.equal(dq[:, D:], want_grads[0][:, D:]) and torch.equal(dbias[1:], want_grads[3][1:])
        assert not dk[:, :D].any() and not dv[:, :D].any()
        assert torch.equal(dk[:, D:], want_grads[1][:, D:]) and torch.equal(dv[:, D:], want_grads[2][:, D:])


# ---- biases that are finite, but so low that an fp32 logit holds nothing else ------------------------

@gpu
@TYPES
@pytest.mark.parametrize("value", [-1e9, -1e10, -1e30])
@pytest.mark.parametrize("case", FORBID_CASES[:1] + FORBID_CASES[2:4], ids=FORBID_IDS[:1] + FORBID_IDS[2:4])
def test_a_very_low_bias_under_large_logits(case, value, dtype):
    """Everything far behind at a very low finite value, logits up to some 200: the first keys of a row are all far behind,
    so the running maximum starts there.  Rows with no other key come out finite, and pass no gradient back: their lse, in
    fp32, does not hold what their probabilities need.

    The reference takes -4000, as above."""
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    q = (q.float() * 50).to(dtype)
    side, B, Tq = buckets.num_buckets // 2, case[0], case[4]
    finite = bias.clone()
    finite[:, side - 1] = -4000.0
    bias[:, side - 1] = value
    first = buckets._side.index(side - 1)
    nk = case[8] or [case[5]] * B
    cut = i64([min(Tq, n - 1 + first) for n in nk])
    live = torch.arange(Tq, device="cuda") < cut.view(-1, 1, 1)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    ref = ref_of(q, k, v, finite, buckets, opts | dict(query_lengths=cut), dout)
    assert_within("lse", torch.where(live, lse, -math.inf), ref["lse"])
    assert_within("out", torch.where(live, out, 0), ref["out"])
    for name, g in zip(GRADS, bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)):
        assert_within(name, g, ref[name])


# ---- what a pass must not look at ------------------------------------------------------------------

@gpu
@TYPES
@pytest.mark.parametrize("val", [math.nan, math.inf])
@pytest.mark.parametrize("case", [
    (2, 8, 2, 64, 8, 500, (32, 128, False), True, None, [3, 8], [100, 77]),        # a padded chunk of new tokens, a cache not yet full
    (1, 2, 2, 96, 40, 200, (32, 128, False), True, None, [21], [90]),
    (2, 16, 4, 128, 150, 400, (32, 128, False), True, None, [101, 0], [30, 5]),
    (1, 4, 1, 64, 1, 1000, (32, 128, False), True, None, None, [637]),
], ids=lambda c: f"B{c[0]}H{c[1]}-{c[2]}D{c[3]}T{c[4]}-{c[5]}")
def test_keys_that_causal_hides_from_every_query(case, val, dtype):
    """A causal cache without key_lengths: what lies behind the last query's position may hold anything."""
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    nq = case[9] or [case[4]] * case[0]
    seen = i64([s + n if n else 0 for s, n in zip(case[10], nq)])
    hidden = torch.arange(case[5], device="cuda") >= seen.view(-1, 1, 1)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    grads = bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)
    k2, v2 = k.masked_fill(hidden, val), v.masked_fill(hidden, val)
    out2, lse2 = bucket_attention(q, k2, v2, bias, buckets, return_lse=True, **opts)
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    for a, b in zip(bucket_attention_backward(dout, q, k2, v2, out, lse, bias, buckets, **opts), grads):
        assert torch.equal(a, b)


@gpu
@TYPES
@pytest.mark.parametrize("D", [40, 64, 33, 5])
@pytest.mark.parametrize("Tq,Tk", [(1, 700), (43, 43), (200, 200)])
def test_an_infinite_key(D, Tq, Tk, dtype):
    """A last key with an infinity in its last channel, which every query turns into -inf: the same as without that key,
    whatever the head's width."""
    b = RelativeBuckets(8, 20)
    q, k, v, bias, _ = inputs(dtype, 2, 2, 2, D, Tq, Tk, b)
    q.view(2, 2, D, Tq)[:, :, -1] = -q.view(2, 2, D, Tq)[:, :, -1].abs() - 0.1
    k.view(2, 2, D, Tk)[:, :, -1, -1] = math.inf
    out, lse = bucket_attention(q, k, v, bias, b, heads=2, return_lse=True)
    ref = ref_of(q, k, v, bias, b, dict(heads=2, kv_heads=2, key_lengths=i64([Tk - 1] * 2), query_lengths=None, query_start=None,
                                        causal=False))
    assert_within("out", out, ref["out"])
    assert_within("lse", lse, ref["lse"])


# ---- state, and other kinds of differentiation -------------------------------------------------------

@gpu
def test_a_validation_pass_before_training():
    """The bucket table is first used under inference_mode, then by a call that autograd records."""
    case = (1, 2, 2, 32, 21, 21, (8, 16, True), False, None, None, None)
    q, k, v, bias, dout, buckets, opts = both(case, torch.float32)
    with torch.inference_mode():
        want = bucket_attention(q, k, v, bias, buckets, **opts)
    with torch.enable_grad():
        leaves = [t.clone().requires_grad_() for t in (q, k, v, bias)]
        out = bucket_attention(*leaves, buckets, **opts)
        out.backward(dout)
    assert torch.equal(out, want) and all(t.grad is not None for t in leaves)


def test_the_table_of_an_unnamed_device_is_the_current_ones(monkeypatch):
    b = RelativeBuckets(8, 18)
    monkeypatch.setattr(attention, "_TABLES", {}, raising=False)
    current = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.Tensor, "to", lambda self, device, *a: (self, device))
    first = b.table("cuda")
    current[0] = 1
    second = b.table("cuda")
    assert first[1] == torch.device("cuda", 0) and second[1] == torch.device("cuda", 1)
    assert b.table(torch.device("cuda", 1)) is second and b.table("cuda:0") is first


@gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    b = RelativeBuckets(8, 20)
    q, k, v, bias, dout = inputs(torch.float32, 1, 1, 1, 32, 16, 16, b)
    out, lse = bucket_attention(q, k, v, bias, b, heads=1, return_lse=True)
    with fwd.dual_level():
        for n in range(4):
            args = [q, k, v, bias]
            args[n] = fwd.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(native.NativeError, match="forward"):
                bucket_attention(*args, b, heads=1)
            with pytest.raises(native.NativeError, match="forward"):
                bucket_attention_backward(dout, *args[:3], out, lse, args[3], b, heads=1)
        with pytest.raises(native.NativeError, match="forward"):
            bucket_attention_backward(fwd.make_dual(dout, dout), q, k, v, out, lse, bias, b, heads=1)
        assert torch.equal(bucket_attention(q, k, v, bias, b, heads=1), out)


@gpu
def test_a_graph_outlives_the_buckets_it_was_captured_with():
    """The table belongs to the buckets' numbers, not to the object: it is not given back while a graph still reads it."""
    b = RelativeBuckets(8, 22)
    q, k, v, bias, _ = inputs(torch.float32, 1, 2, 2, 32, 50, 50, b)
    want = bucket_attention(q, k, v, bias, b, heads=2)
    size = b.table("cuda").numel()
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        out = bucket_attention(q, k, v, bias, b, heads=2)
    del b
    others = [torch.full((size,), 7, device="cuda", dtype=torch.int32) for _ in range(64)]      # would take its place
    for _ in range(3):
        out.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del others


# ---- C entries -------------------------------------------------------------------------------------

def test_c_entries_refuse_negative_and_endless_strides():
    L = native.lib()
    names = [n + s for n in ("q", "k", "v", "out") for s in ("_bstride", "_cstride")]
    more = [n + s for n in ("dout", "dq", "dk", "dv") for s in ("_bstride", "_cstride")]
    room = dict(workspace=4096, workspace_bytes=1 << 40)
    for n in names:
        assert L.vk_bucket_attention(C.byref(_args(**{n: -100}, **room)), None) == -1, n
    for n in names + more:
        assert L.vk_bucket_attention_backward(C.byref(_args(**{n: -100}, **room)), None) == -1, n
    for n in ("q", "out", "dout", "dq", "dk", "dv"):                           # a sum of them would wrap
        assert L.vk_bucket_attention_backward(C.byref(_args(**{n + "_cstride": 1 << 62}, **room)), None) == -1, n
        assert L.vk_bucket_attention_backward(C.byref(_args(**{n + "_bstride": 1 << 62}, **room)), None) == -1, n
