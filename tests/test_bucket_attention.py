"""Attention with a bucketed relative position bias and its backward pass against the definition in 64 bits.

Tolerances are bounds on the rounding errors, derived per element from the inputs.  With u = 2^-24 (half a step
of fp32) and r = half a step of the tensors' type (bf16 2^-8; 0 for what stays fp32 inside):

* a logit is off by at most e_s = ((D + 4) u) scale sum |q||k| + 4 u |bias| + 2 u |lse| (products, sums, the bias, the
  subtraction of the log-sum-exp), so a probability by a factor of 1 +- (2 e_s + 8 u): its own logit and the normaliser;
* sums of n terms add n u of the sum of their magnitudes;
* bf16: probabilities and logit gradients are rounded once where they enter a product (r of each term's magnitude),
  results once when they are stored, and the saved output inside delta = dout . out once as well.
"""
import ctypes as C
import math

import pytest
import torch

from vits_amd import attention, native
from vits_amd.attention import RelativeBuckets, bucket_attention, bucket_attention_backward

gpu = pytest.mark.gpu
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, bias, buckets, heads, kv_heads, nk, nq, start, causal, dout=None):
    """{name: (value, bound)} in 64 bits on the CPU, whole matrices."""
    dt = q.dtype
    r = half_step(dt) if dt != torch.float32 else 0.0
    B, C_, Tq = q.shape
    D, Tk, G = C_ // heads, k.shape[2], heads // kv_heads
    cpu = lambda t: t.detach().cpu().double()
    q, k, v = (cpu(t).reshape(B, -1, D, t.shape[2]) for t in (q, k, v))
    nk = torch.full((B,), Tk) if nk is None else nk.cpu().clamp(0, Tk)
    nq = torch.full((B,), Tq) if nq is None else nq.cpu().clamp(0, Tq)
    start = torch.zeros(B, dtype=torch.int64) if start is None else start.cpu()
    j, i = torch.arange(Tk), torch.arange(Tq)
    off = j.view(1, 1, Tk) - (i.view(1, Tq, 1) + start.view(B, 1, 1))
    ok = (j.view(1, 1, Tk) < nk.view(B, 1, 1)) & (i.view(1, Tq, 1) < nq.view(B, 1, 1))
    if causal:
        ok = ok & (off <= 0)
    live_k, live_q = (j.view(1, Tk) < nk.view(B, 1)).view(B, 1, 1, Tk), (i.view(1, Tq) < nq.view(B, 1)).view(B, 1, 1, Tq)
    q = q.masked_fill(~live_q, 0)                       # what is behind a length is not part of the definition
    k, v = k.masked_fill(~live_k, 0), v.masked_fill(~live_k, 0)
    kg, vg = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    scale = D ** -0.5
    s = q.transpose(2, 3) @ kg * scale
    mag = q.abs().transpose(2, 3) @ kg.abs() * scale
    if bias is not None:
        lut = torch.tensor([buckets.bucket_of(o) for o in range(-buckets.max_distance, buckets.max_distance + 1)])
        where = lut[off.clamp(-buckets.max_distance, buckets.max_distance) + buckets.max_distance]
        bv = cpu(bias)[:, where].transpose(0, 1)
        s = s + bv
        mag = mag + bv.abs() / (D + 4) * 4
    okh = ok.unsqueeze(1).expand(B, heads, Tq, Tk)
    s = s.masked_fill(~okh, -math.inf)
    lse = torch.logsumexp(s, -1) if Tk else torch.full(s.shape[:-1], -math.inf, dtype=torch.float64)
    some = lse > -math.inf
    p = torch.exp(s - lse.masked_fill(~some, 0).unsqueeze(-1)).masked_fill(~okh, 0)
    e_s = (D + 4) * U * mag.amax((-1, -2), keepdim=True) + 2 * U * lse.masked_fill(~some, 0).abs().unsqueeze(-1) if Tk and Tq \
        else torch.zeros(B, heads, 1, 1, dtype=torch.float64)
    rel = 2 * e_s + 8 * U                                # of a probability
    store = lambda x, b, dtype: (x, b + half_step(dtype) * (x.abs() + b) + 1e-30)
    out = (p @ vg.transpose(2, 3)).transpose(2, 3)       # [B, H, D, Tq]
    b_out = ((p * (rel + r + Tk * U)) @ vg.abs().transpose(2, 3)).transpose(2, 3)
    flat = lambda x: x.reshape(B, -1, x.shape[-1])
    res = {"out": store(flat(out), flat(b_out), dt),
           "lse": store(lse, (rel + Tk * U).expand(B, heads, Tq, 1).squeeze(-1), torch.float32)}
    if dout is None:
        return res
    do = cpu(dout).reshape(B, heads, D, Tq).masked_fill(~live_q, 0)
    delta = (do * out).sum(2).unsqueeze(-1)
    dp = do.transpose(2, 3) @ vg
    ds = p * (dp - delta)
    e_d = (D + 4) * U * (do.abs().transpose(2, 3) @ vg.abs()) \
        + (((D + 4) * U + half_step(dt)) * (do.abs() * out.abs()).sum(2) + (do.abs() * b_out).sum(2)).unsqueeze(-1)
    b_ds = ds.abs() * rel + p * e_d
    sum_heads = lambda x: x.reshape(B, kv_heads, G, D, Tk).sum(2)
    dq = kg @ ds.transpose(2, 3) * scale
    b_dq = kg.abs() @ (b_ds + ds.abs() * (r + Tk * U)).transpose(2, 3) * scale
    dk = sum_heads(q @ ds * scale)
    b_dk = sum_heads(q.abs() @ (b_ds + ds.abs() * (r + G * Tq * U)) * scale)
    dv = sum_heads(do @ p)
    b_dv = sum_heads(do.abs() @ (p * (rel + r + G * Tq * U)))
    res |= {"dq": store(flat(dq), flat(b_dq), dt), "dk": store(flat(dk), flat(b_dk), dt), "dv": store(flat(dv), flat(b_dv), dt)}
    if bias is not None:
        dbias, b = torch.zeros(heads, buckets.num_buckets, dtype=torch.float64), torch.zeros(heads, buckets.num_buckets, dtype=torch.float64)
        for h in range(heads):
            dbias[h].index_add_(0, where.expand(B, Tq, Tk).reshape(-1), ds[:, h].reshape(-1))
            # a sum over n terms in some order: n u of the magnitudes, n at most the rows' length times their number
            b[h].index_add_(0, where.expand(B, Tq, Tk).reshape(-1), (b_ds + ds.abs() * (Tk + Tq + 64 * B) * U)[:, h].reshape(-1))
        res["dbias"] = store(dbias, b, torch.float32)
    return res


def assert_within(name, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(got[~fine], value[~fine]), name
    off = (got - value)[fine].abs() - bound[fine]
    assert not torch.isnan(got[fine]).any(), name
    if off.numel():
        worst = off.argmax()
        assert off.max() <= 0, (name, float(got[fine][worst]), float(value[fine][worst]), float(bound[fine][worst]))


def inputs(dtype, B, H, Hk, D, Tq, Tk, buckets, seed=0, fused=False):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    if fused:
        qkv = rnd(B, (H + 2 * Hk) * D, Tk).to(dtype).cuda()
        q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:]
    else:
        q, k, v = (rnd(B, n * D, t).to(dtype).cuda() for n, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
    bias = rnd(H, buckets.num_buckets).cuda() if buckets is not None else None
    return q, k, v, bias, rnd(B, H * D, Tq).to(dtype).cuda()


def i64(x):
    return None if x is None else torch.tensor(x, device="cuda", dtype=torch.int64)


BIDIR, WIDE, SMALL = (32, 128, True), (16, 300, True), (8, 20, True)
# B, H, Hk, D, Tq, Tk, buckets (num, distance, bidirectional), causal, nk, nq, start
CASES = [
    (1, 2, 2, 96, 43, 43, BIDIR, False, None, None, None),                # one sentence of the text encoder
    (1, 1, 1, 1, 1, 1, SMALL, False, None, None, None),
    (2, 3, 1, 40, 65, 200, SMALL, False, [200, 131], [65, 64], [135, 67]),
    (3, 4, 4, 32, 257, 257, WIDE, False, [257, 0, 100], [257, 0, 100], None),     # an item of length zero
    (2, 4, 2, 64, 129, 129, (32, 128, False), True, None, None, None),
    (2, 4, 1, 128, 300, 300, (32, 128, False), True, [300, 77], [300, 77], None),
    (1, 2, 2, 80, 31, 33, None, False, None, None, None),                 # no bias
    (2, 8, 2, 128, 1, 1000, (32, 128, False), True, [1000, 63], None, [999, 62]),  # one new token over a cache
    (2, 4, 4, 64, 5, 321, (32, 128, False), True, [321, 64], None, [316, 59]),
    (2, 2, 2, 64, 70, 70, (32, 128, False), True, [70, 70], None, [-40, 500]),     # rows that see nothing; all in sight
    (1, 12, 3, 72, 97, 513, BIDIR, False, [500], [96], [200]),
    (1, 1, 1, 33, 640, 640, (64, 1024, True), False, None, None, None),
]
IDS = [f"B{c[0]}H{c[1]}-{c[2]}D{c[3]}T{c[4]}-{c[5]}{'c' if c[7] else ''}" for c in CASES]


def both(case, dtype, seed=0, **kw):
    B, H, Hk, D, Tq, Tk, bk, causal, nk, nq, start = case
    buckets = RelativeBuckets(bk[0], bk[1], bidirectional=bk[2]) if bk else None
    q, k, v, bias, dout = inputs(dtype, B, H, Hk, D, Tq, Tk, buckets, seed, **kw)
    opts = dict(heads=H, kv_heads=Hk, key_lengths=i64(nk), query_lengths=i64(nq), query_start=i64(start), causal=causal)
    return q, k, v, bias, dout, buckets, opts


def ref_of(q, k, v, bias, buckets, opts, dout=None):
    return reference(q, k, v, bias, buckets, opts["heads"], opts["kv_heads"], opts["key_lengths"], opts["query_lengths"],
                     opts["query_start"], opts["causal"], dout)


# ---- on the CPU ------------------------------------------------------------------------------------

@pytest.mark.parametrize("nb,far", [(32, 128), (16, 64), (8, 20), (64, 1024), (4, 3)])
def test_bucket_map_follows_its_definition(nb, far):
    """Distance n >= single is in range r iff single * (far / single)^(r / m) <= n < the next one's; borders in exact
    rationals (both sides to the m-th power)."""
    for bidir in (True, False):
        b = RelativeBuckets(nb, far, bidirectional=bidir)
        side = nb // 2 if bidir else nb
        single, m = side // 2, side - side // 2
        last = -1
        for n in range(0, far + 40):
            got = b.bucket_of(-n)
            assert got >= last, "monotone in the distance"
            last = got
            if n < single:
                assert got == n
            else:
                r = got - single
                nn = min(n, far)
                assert nn ** m * single ** r >= far ** r * single ** m
                assert r == m - 1 or nn ** m * single ** (r + 1) < far ** (r + 1) * single ** m
            assert b.bucket_of(n) == ((got + side if n else got) if bidir else (0 if n else got))
        assert b.bucket_of(-far) == side - 1


@pytest.mark.parametrize("bad", [dict(num_buckets=3), dict(num_buckets=31), dict(num_buckets=32, max_distance=8),
                                 dict(max_distance=1025), dict(num_buckets=1, bidirectional=False)])
def test_bucket_map_refusals(bad):
    with pytest.raises(ValueError):
        RelativeBuckets(**bad)


def _args(**kw):
    a = native.BucketAttentionArgs()
    for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "dbias", "bias", "bucket_of"):
        setattr(a, n, 4096)
    a.batch, a.heads, a.kv_heads, a.head_dim, a.queries, a.keys = 2, 4, 2, 64, 100, 100
    for n in ("q", "out", "dout", "dq"):
        setattr(a, n + "_bstride", 25600), setattr(a, n + "_cstride", 100)
    for n in ("k", "v", "dk", "dv"):
        setattr(a, n + "_bstride", 12800), setattr(a, n + "_cstride", 100)
    a.has_bias, a.buckets, a.max_distance, a.scale, a.dtype = 1, 32, 128, 0.125, native.DTYPE_F32
    for n, val in kw.items():
        setattr(a, n, val)
    return a


@pytest.mark.parametrize("bad,code", [
    (dict(heads=3), -1), (dict(kv_heads=0), -1), (dict(queries=-1), -1), (dict(batch=-1), -1), (dict(head_dim=0), -2),
    (dict(head_dim=129), -2), (dict(dtype=2), -2), (dict(buckets=0), -2), (dict(max_distance=1025), -2),
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(keys=(1 << 28) + 1), -2), (dict(q=0), -1),
    (dict(k=0), -1), (dict(bias=0), -1), (dict(bucket_of=0), -1)])
def test_c_entries_refuse_bad_arguments(bad, code):
    L = native.lib()
    a = _args(**bad)
    for entry in (L.vk_bucket_attention, L.vk_bucket_attention_backward):
        assert entry(C.byref(a), None) == code
        assert L.vk_last_error().decode().startswith("vk_bucket_attention")


def test_c_entries_refuse_missing_outputs_overlaps_and_short_workspaces():
    L = native.lib()
    E = lambda f, a: f(C.byref(a), None)
    assert E(L.vk_bucket_attention, _args(out=0)) == -1
    assert E(L.vk_bucket_attention, _args(out_cstride=99)) == -1
    assert E(L.vk_bucket_attention, _args(out_bstride=100)) == -1
    for n in ("dq", "dk", "dv", "dbias", "dout", "lse"):
        assert E(L.vk_bucket_attention_backward, _args(**{n: 0})) == -1, n
    for n in ("dq", "dk", "dv"):
        assert E(L.vk_bucket_attention_backward, _args(**{n + "_cstride": 99})) == -1, n
    assert L.vk_bucket_attention(None, None) == -1
    small = _args(queries=1, keys=1000, k_cstride=1000, v_cstride=1000)        # shares the keys out
    need = L.vk_bucket_attention_workspace_bytes(C.byref(small))
    assert need > 0
    small.workspace, small.workspace_bytes = 4096, need - 4
    assert E(L.vk_bucket_attention, small) == -4
    a = _args()
    need = L.vk_bucket_attention_backward_workspace_bytes(C.byref(a))
    a.workspace, a.workspace_bytes = 4096, need - 4
    assert need > 0 and E(L.vk_bucket_attention_backward, a) == -4
    assert L.vk_bucket_attention_workspace_bytes(C.byref(_args(heads=3))) == -1
    assert L.vk_bucket_attention_workspace_bytes(C.byref(_args(batch=1 << 20, heads=16, kv_heads=2))) == -2    # more heads than a grid holds
    a.workspace, a.workspace_bytes = 4104, need
    assert E(L.vk_bucket_attention_backward, a) == -1                          # not 16-byte aligned
    for bad in (0.0, -1.0):
        assert E(L.vk_bucket_attention, _args(scale=bad)) == -1


def test_nothing_to_do_is_accepted():
    L = native.lib()
    for none in (dict(batch=0), dict(queries=0), dict(keys=0)):
        assert L.vk_bucket_attention_workspace_bytes(C.byref(_args(**none))) == 0
        assert L.vk_bucket_attention_backward_workspace_bytes(C.byref(_args(**none))) >= 0
    assert L.vk_bucket_attention(C.byref(_args(batch=0, q=0, k=0, v=0, out=0, lse=0)), None) == 0
    assert L.vk_bucket_attention(C.byref(_args(queries=0, q=0, out=0, lse=0)), None) == 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 64, 8)
    with pytest.raises(native.NativeError):
        bucket_attention(q, q, q, heads=1)


# ---- on the GPU ------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_and_backward(case, dtype):
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    assert_within("out", out, ref["out"])
    assert_within("lse", lse, ref["lse"])
    grads = bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)
    for name, g in zip(("dq", "dk", "dv", "dbias"), grads):
        if g is not None:
            assert_within(name, g, ref[name])
    again = bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again)), "the same inputs give the same bits"
    assert torch.equal(out, bucket_attention(q, k, v, bias, buckets, **opts))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_workgroups(dtype):
    """Enough heads and queries for the widest query tiles, and for heads dealt over the XCDs unevenly."""
    case = (17, 16, 8, 64, 520, 520, (32, 128, False), True, [520 - 31 * i for i in range(17)], [520 - 31 * i for i in range(17)], None)
    q, k, v, bias, dout, buckets, opts = both(case, dtype, fused=True)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    assert_within("out", out, ref["out"])
    assert_within("lse", lse, ref["lse"])
    for name, g in zip(("dq", "dk", "dv", "dbias"), bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)):
        assert_within(name, g, ref[name])


SHARED = [
    (1, 16, 1, 128, 300, 300, (32, 128, False), True, None, None, None),          # queries of 16 heads in shares, causal
    (2, 2, 2, 96, 500, 333, BIDIR, False, [333, 0], [500, 411], [3, 0]),          # shares of one head's queries, an empty item
    (1, 8, 2, 64, 257, 255, SMALL, False, [251], [130], None),                    # shares beyond the length
    (3, 6, 2, 72, 129, 129, None, True, [129, 1, 64], [129, 1, 64], None),
    (33, 4, 4, 32, 1, 70, (32, 128, False), True, [70 - i for i in range(33)], None, [69 - i for i in range(33)]),   # tokens of many heads
    (1, 2, 2, 64, 60, 1500, BIDIR, False, [1489], None, [700]),                   # few rows, long: wide tiles, shared keys
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", SHARED, ids=[f"B{c[0]}H{c[1]}-{c[2]}D{c[3]}T{c[4]}-{c[5]}" for c in SHARED])
def test_shares_of_the_other_axis(case, dtype):
    test_forward_and_backward(case, dtype)


@gpu
@pytest.mark.parametrize("Tq,Tk", [(0, 5), (5, 0), (0, 0)])
def test_empty_lengths(Tq, Tk):
    b = RelativeBuckets(8, 20)
    q, k, v, bias, dout = inputs(torch.float32, 2, 2, 2, 32, Tq, Tk, b)
    out, lse = bucket_attention(q, k, v, bias, b, heads=2, return_lse=True)
    assert out.shape == (2, 64, Tq) and not out.any() and (lse == -math.inf).all()
    dq, dk, dv, dbias = bucket_attention_backward(dout, q, k, v, out, lse, bias, b, heads=2)
    assert dq.shape == q.shape and dk.shape == k.shape and not dq.any() and not dk.any() and not dv.any() and not dbias.any()
    q0, k0, v0, _, d0 = inputs(torch.float32, 0, 2, 2, 32, 4, 4, b)
    out, lse = bucket_attention(q0, k0, v0, bias, b, heads=2, return_lse=True)
    assert out.shape == (0, 64, 4)
    assert not bucket_attention_backward(d0, q0, k0, v0, out, lse, bias, b, heads=2)[3].any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_padding_may_hold_anything(dtype):
    """NaN and infinities behind the lengths, in every input, change no bit of the result."""
    case = (3, 4, 2, 64, 150, 150, BIDIR, False, [150, 0, 37], [150, 0, 37], None)
    q, k, v, bias, dout, buckets, opts = both(case, dtype)
    lens = opts["key_lengths"]
    dirty = lambda t, val: torch.where(torch.arange(150, device="cuda") >= lens.view(-1, 1, 1), torch.tensor(val, dtype=dtype, device="cuda"), t)
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    grads = bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)
    for val in (math.nan, math.inf, torch.finfo(dtype).min):
        q2, k2, v2, d2, o2 = (dirty(t, val) for t in (q, k, v, dout, out))
        got, lse2 = bucket_attention(q2, k2, v2, bias, buckets, return_lse=True, **opts)
        assert torch.equal(got, out) and torch.equal(lse2, lse)
        lse2 = torch.where(torch.arange(150, device="cuda") >= lens.view(-1, 1, 1), torch.tensor(val, device="cuda").float(), lse)
        for a, b in zip(bucket_attention_backward(d2, q2, k2, v2, o2, lse2, bias, buckets, **opts), grads):
            assert torch.equal(a, b)
    pad = torch.arange(150, device="cuda").view(1, 1, -1) >= lens.view(-1, 1, 1)
    assert not out.masked_select(pad).any() and all(not g.masked_select(pad).any() for g in grads[:3])


@gpu
def test_lengths_beyond_the_tensors_are_clamped():
    case = (2, 2, 2, 32, 40, 40, SMALL, False, [400, -3], [41, 40], None)
    q, k, v, bias, dout, buckets, opts = both(case, torch.float32)
    out = bucket_attention(q, k, v, bias, buckets, **opts)
    opts["key_lengths"], opts["query_lengths"] = i64([40, 0]), None
    assert torch.equal(out, bucket_attention(q, k, v, bias, buckets, **opts))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_views_of_larger_buffers(dtype):
    """Slices of a fused projection that start at an odd position, and a cache with room to grow."""
    b = RelativeBuckets(16, 64)
    g = torch.Generator().manual_seed(3)
    big = torch.randn(2, 5 * 64, 301, generator=g).to(dtype).cuda()
    view = big[:, 64:256, 3:120]
    q, k, v = view[:, :64], view[:, 64:128], view[:, 128:]
    bias = torch.randn(2, 16, generator=g).cuda()
    dout = torch.randn(2, 64, 240, generator=g).to(dtype).cuda()[:, :, 1:118]
    out, lse = bucket_attention(q, k, v, bias, b, heads=2, return_lse=True)
    c = [t.contiguous() for t in (q, k, v, dout)]
    out_c, lse_c = bucket_attention(*c[:3], bias, b, heads=2, return_lse=True)
    assert torch.equal(out, out_c) and torch.equal(lse, lse_c)
    for x, y in zip(bucket_attention_backward(dout, q, k, v, out, lse, bias, b, heads=2),
                    bucket_attention_backward(c[3], *c[:3], out, lse, bias, b, heads=2)):
        assert torch.equal(x, y)


@gpu
def test_saved_output_and_gradient_in_another_order():
    """out and dout with the channels dense, as a transposed result of other code has them."""
    b = RelativeBuckets(8, 20)
    q, k, v, bias, dout = inputs(torch.float32, 2, 1, 1, 48, 37, 37, b)
    out, lse = bucket_attention(q, k, v, bias, b, heads=1, return_lse=True)
    turned = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert turned(out).stride(2) != 1
    for x, y in zip(bucket_attention_backward(dout, q, k, v, out, lse, bias, b, heads=1),
                    bucket_attention_backward(turned(dout), q, k, v, turned(out), lse, bias, b, heads=1)):
        assert torch.equal(x, y)


@gpu
def test_rows_around_the_outputs_stay_as_they_were():
    """Outputs written into views: nothing outside them is touched."""
    b = RelativeBuckets(8, 20)
    q, k, v, bias, dout = inputs(torch.bfloat16, 2, 2, 2, 40, 77, 77, b)
    room = torch.full((2, 100, 90), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.empty(2, 2, 77, device="cuda")
    common = dict(heads=2, kv_heads=2, scale=40 ** -0.5)
    native.bucket_attention(q, k, v, room[:, 8:88, 5:82], lse, bias, b.table("cuda"), **common)
    want = bucket_attention(q, k, v, bias, b, heads=2)
    assert torch.equal(room[:, 8:88, 5:82], want)
    room[:, 8:88, 5:82] = 7.0
    assert (room == 7.0).all()
    rooms = [torch.full((2, 90, 91), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    dbias = torch.empty_like(bias)
    native.bucket_attention_backward(dout, q, k, v, want, lse, *(t[:, 5:85, 3:80] for t in rooms), bias, b.table("cuda"), dbias, **common)
    for t, w in zip(rooms, bucket_attention_backward(dout, q, k, v, want, lse, bias, b, heads=2)):
        assert torch.equal(t[:, 5:85, 3:80], w)
        t[:, 5:85, 3:80] = 7.0
        assert (t == 7.0).all()


@gpu
def test_offsets_beyond_32_bits():
    """A cache whose last channel rows start behind 2^31 elements."""
    b = RelativeBuckets(32, 128, bidirectional=False)
    cache = torch.empty(1, 256, 1 << 24, device="cuda", dtype=torch.bfloat16)
    q, k, v, bias, dout = inputs(torch.bfloat16, 1, 1, 1, 128, 70, 300, b)
    cache[:, :128, :300], cache[:, 128:, :300] = k, v
    opts = dict(heads=1, query_start=i64([230]), causal=True)
    out, lse = bucket_attention(q, k, v, bias, b, return_lse=True, **opts)
    kc, vc = cache[:, :128, :300], cache[:, 128:, :300]
    assert torch.equal(out, bucket_attention(q, kc, vc, bias, b, **opts))
    for x, y in zip(bucket_attention_backward(dout, q, k, v, out, lse, bias, b, **opts),
                    bucket_attention_backward(dout, q, kc, vc, out, lse, bias, b, **opts)):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_large_logits(spread):
    """Logits of a few hundred: the running maximum keeps every exponent in range."""
    case = (1, 2, 2, 64, 200, 200, BIDIR, False, None, None, None)
    q, k, v, bias, dout, buckets, opts = both(case, torch.float32)
    q, bias = q * spread, bias * spread
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    assert_within("out", out, ref["out"])
    assert_within("lse", lse, ref["lse"])
    for name, g in zip(("dq", "dk", "dv", "dbias"), bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)):
        assert_within(name, g, ref[name])


@gpu
def test_autograd_and_differences():
    """Gradients through autograd equal the explicit backward pass, and along random directions the derivative of the
    64-bit definition by central differences."""
    case = (2, 4, 2, 48, 61, 61, SMALL, False, [61, 20], [61, 20], None)
    q, k, v, bias, dout, buckets, opts = both(case, torch.float32)
    with torch.enable_grad():
        leaves = [t.clone().requires_grad_() for t in (q, k, v, bias)]
        out = bucket_attention(*leaves, buckets, **opts)
        got = torch.autograd.grad(out, leaves, dout)
        total = bucket_attention(*leaves, buckets, **opts).sum()        # an expanded gradient
        total.backward()
    out, lse = bucket_attention(q, k, v, bias, buckets, return_lse=True, **opts)
    for a, b in zip(got, bucket_attention_backward(dout, q, k, v, out, lse, bias, buckets, **opts)):
        assert torch.equal(a, b)
    ones = bucket_attention_backward(torch.ones_like(dout), q, k, v, out, lse, bias, buckets, **opts)
    assert all(torch.equal(leaf.grad, b) for leaf, b in zip(leaves, ones))
    ref = ref_of(q, k, v, bias, buckets, opts, dout)
    at = [t.cpu().double() for t in (q, k, v, bias)]
    w = dout.cpu().double()
    f = lambda *t: float((ref_of(*t, buckets, opts)["out"][0] * w).sum())
    g = torch.Generator().manual_seed(11)
    for n, name in enumerate(("dq", "dk", "dv", "dbias")):
        step = torch.randn(at[n].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        moved = [[x + (s * eps * step if m == n else 0) for m, x in enumerate(at)] for s in (1, -1)]
        diff = (f(*moved[0]) - f(*moved[1])) / (2 * eps)
        along = float((got[n].cpu().double() * step).sum())
        # third derivatives are below 1e3 here: eps^2 * 1e3, and the bound of every entry along the step
        assert abs(diff - along) <= float((ref[name][1] * step.abs()).sum()) + 1e-7 * max(1.0, abs(diff))


@gpu
def test_streams_and_graphs():
    """Calls on another stream, captured and replayed with eager work between, and two graphs that replay in turn."""
    b = RelativeBuckets(32, 128, bidirectional=False)
    b.table("cuda")
    sets = [inputs(torch.bfloat16, 1, 4, 2, 64, t, t, b, seed=t) for t in (1, 70, 333)]

    def step(q, k, v, bias, dout):
        out, lse = bucket_attention(q, k, v, bias, b, heads=4, kv_heads=2, causal=True, return_lse=True)
        return (out, lse, *bucket_attention_backward(dout, q, k, v, out, lse, bias, b, heads=4, kv_heads=2, causal=True))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    graphs = []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(*s)
        graphs.append((gr, res))
    for _ in range(3):
        for (gr, res), s, w in zip(graphs, sets, want):
            for t in res:
                t.fill_(3.0)
            gr.replay()
            step(*sets[1])
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(res, w))


@gpu
def test_capture_under_autograd_is_refused():
    b = RelativeBuckets(8, 20)
    q, k, v, bias, _ = inputs(torch.float32, 1, 1, 1, 32, 16, 16, b)
    bucket_attention(q, k, v, bias, b, heads=1)
    torch.cuda.synchronize()
    fresh = RelativeBuckets(8, 20)
    gr = torch.cuda.CUDAGraph()
    with torch.enable_grad(), torch.cuda.graph(gr):
        with pytest.raises(native.NativeError, match="captured"):
            bucket_attention(q.requires_grad_(), k, v, bias, b, heads=1)
        with pytest.raises(native.NativeError, match="before the capture"):
            bucket_attention(q.detach(), k, v, bias, fresh, heads=1)


@gpu
def test_refusals():
    b = RelativeBuckets(8, 20)
    q, k, v, bias, dout = inputs(torch.float32, 2, 4, 2, 32, 16, 24, b)
    ok = dict(heads=4, kv_heads=2)
    out, lse = bucket_attention(q, k, v, bias, b, return_lse=True, **ok)
    bad = [
        (dict(q=q.half(), k=k.half(), v=v.half()), {}), (dict(k=k.bfloat16()), {}), (dict(q=q[0]), {}), (dict(v=v[:, :, :20]), {}),
        (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), {}), (dict(bias=None), {}), (dict(bias=bias[:, :4]), {}),
        (dict(bias=bias.double()), {}), (dict(k=k[:, :32], v=v[:, :32]), {}), ({}, dict(heads=3)), ({}, dict(kv_heads=3)),
        ({}, dict(key_lengths=torch.tensor([1, 2], device="cuda", dtype=torch.int32))), ({}, dict(key_lengths=torch.tensor([1, 2]))),
        ({}, dict(query_start=i64([1]))), ({}, dict(scale=math.inf)), (dict(k=k.cpu(), v=v.cpu()), {}),
    ]
    for tensors, opts in bad:
        t = dict(q=q, k=k, v=v, bias=bias) | tensors
        with pytest.raises(ValueError):
            bucket_attention(t["q"], t["k"], t["v"], t["bias"], b, **(ok | opts))
    for args in ((dout[:, :, :3], out, lse), (dout.bfloat16(), out, lse), (dout, out[:, :64], lse), (dout, out, lse.double()),
                 (dout, out, lse[:, :2])):
        with pytest.raises(ValueError):
            bucket_attention_backward(args[0], q, k, v, args[1], args[2], bias, b, **ok)
    wide = torch.zeros(1, 129, 4, device="cuda")
    with pytest.raises(ValueError):
        bucket_attention(wide, wide, wide, heads=1)
