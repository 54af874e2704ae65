"""Cases of the transformer-block operators: attention with a learned relative position bias by
buckets (whole sequences and single tokens), its backward pass, and the block norm (the norm after a
block, its gate and residual scale, the residual sum and the norm before the next block) with its
backward pass.  Tensors are channel-major [batch, channels, time] as everywhere in this package;
batches are padded, ``lengths`` say how far each item goes."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ----------------------------------------------------------------------------------------

def _att(op, name, dtype, batch, heads, kv_heads, dim, queries, keys, *, causal=False, ragged=False, last=False,
         buckets=32, distance=128):
    c = dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, queries=queries, keys=keys,
             causal=causal, ragged=ragged, last=last, buckets=buckets, distance=distance)
    return dict(c, name=name) if name else c


def _norm(op, name, dtype, batch, channels, length, *, norm="layer", gate="full", ragged=False):
    c = dict(op=op, dtype=dtype, batch=batch, channels=channels, length=length, norm=norm, gate=gate, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one short sentence through one layer of the text encoder (2 heads of 96, 43 tokens): latency
        _att("attend", "attend_f32_sentence", "f32", 1, 2, 2, 96, 43, 43),
        # a padded batch of long texts at the text encoder's width
        _att("attend", "attend_f32_batch", "f32", 16, 2, 2, 96, 1001, 1001, ragged=True),
        # documents of odd length, every position sees every other
        _att("attend", "attend_bf16_long", "bf16", 4, 8, 8, 64, 8191, 8191),
        # a causal token model with shared key and value heads, padded batch
        _att("attend", "attend_bf16_causal", "bf16", 8, 16, 4, 128, 2048, 2048, causal=True, ragged=True),
        # one new token per item over a cache of 16384 positions
        _att("attend", "attend_bf16_token", "bf16", 16, 16, 4, 128, 1, 16384, causal=True, ragged=True, last=True),
        # training on one short sentence: latency
        _att("attend_grad", "attend_grad_f32_sentence", "f32", 1, 2, 2, 96, 43, 43),
        # training on a padded batch at the text encoder's width
        _att("attend_grad", "attend_grad_f32_batch", "f32", 16, 2, 2, 96, 697, 697, ragged=True),
        # training the causal token model
        _att("attend_grad", "attend_grad_bf16_causal", "bf16", 2, 16, 4, 128, 4095, 4095, causal=True),
        # the norms around one block: one sentence, and a large batch with a gate per item and channel
        _norm("norm", "norm_f32_sentence", "f32", 1, 192, 43),
        _norm("norm", "norm_bf16_batch", "bf16", 8, 1024, 4096, norm="rms", gate="item"),
        # their gradients: the text encoder's width, and a wide odd batch with a gate per position
        _norm("norm_grad", "norm_grad_f32_batch", "f32", 16, 192, 862, gate="item", ragged=True),
        _norm("norm_grad", "norm_grad_bf16_batch", "bf16", 8, 1024, 2047, ragged=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend_grad", "attend_grad", "norm", "norm_grad"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("norm", "norm_grad"):
        while True:
            b, c, t = _log_int(rng, 1, 16), _log_int(rng, 64, 2048), _log_int(rng, 1, 8192)
            if b * c * t <= 16_000_000:
                break
        return _norm(op, None, dtype, b, c, t, norm=rng.choice(["layer", "rms"]), gate=rng.choice(["full", "item"]),
                     ragged=rng.random() < 0.5)
    dim = rng.choice([32, 40, 64, 80, 96, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    buckets, distance = rng.choice([(32, 128), (16, 64), (32, 256), (8, 20)])
    ragged = rng.random() < 0.5
    if op == "attend" and rng.random() < 0.33:      # new tokens over a cache
        while True:
            b, t = _log_int(rng, 1, 32), _log_int(rng, 64, 32768)
            if b * kv * dim * t <= 130_000_000:
                break
        return _att(op, None, dtype, b, heads, kv, dim, rng.choice([1, 1, 1, 2, 5]), t, causal=True, ragged=ragged,
                    last=True, buckets=buckets, distance=distance)
    cap = {"attend": {"f32": 2e10, "bf16": 1e11}, "attend_grad": {"f32": 8e9, "bf16": 2.5e10}}[op][dtype]
    while True:
        b, t = _log_int(rng, 1, 16), _log_int(rng, 1, 8192 if op == "attend" else 4096)
        if b * heads * dim * t * t <= cap:
            break
    return _att(op, None, dtype, b, heads, kv, dim, t, t, causal=rng.random() < 0.5, ragged=ragged, buckets=buckets,
                distance=distance)


def _lengths(case, full):
    """The items' lengths: from the full one down to a third of it, the same for every seed but for their order."""
    b = case["batch"]
    if not case["ragged"]:
        return [full] * b
    return [full - (full * 2 // 3) * i // max(1, b - 1) for i in range(b)]


# ---- inputs ---------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    s = {"case": case}
    b = case["batch"]
    if case["op"] in ("norm", "norm_grad"):
        c, t = case["channels"], case["length"]
        order = torch.randperm(b, generator=gen, device=dev)
        s["lengths"] = torch.tensor(_lengths(case, t), device=dev, dtype=torch.int64)[order] if case["ragged"] else None
        s["y"] = (rnd(b, c, t) * 1.5 + 0.2).to(dt)
        s["gate"] = (rnd(b, c, t if case["gate"] == "full" else 1) * 0.5 + 1).to(dt)
        s["scale"] = rnd(c) * 0.1 + 0.3
        s["post"] = (rnd(c) * 0.2 + 1, rnd(c) * 0.1 if case["norm"] == "layer" else None)
        s["pre"] = (rnd(c) * 0.2 + 1, rnd(c) * 0.1 if case["norm"] == "layer" else None)
        if case["op"] == "norm":
            s["x"] = rnd(b, c, t).to(dt)
        else:
            s["h"], s["dh"], s["dn"] = rnd(b, c, t).to(dt), rnd(b, c, t).to(dt), rnd(b, c, t).to(dt)
        return s
    h, hk, d, tq, tk = (case[n] for n in ("heads", "kv_heads", "dim", "queries", "keys"))
    order = torch.randperm(b, generator=gen, device=dev)
    nk = torch.tensor(_lengths(case, tk), device=dev, dtype=torch.int64)[order]
    if case["last"]:                                      # new tokens at the end of each item's cache
        s["start"], s["nq"] = nk - tq, None
        s["q"] = rnd(b, h * d, tq).to(dt)
        s["k"], s["v"] = rnd(b, hk * d, tk).to(dt), rnd(b, hk * d, tk).to(dt)
    else:                                                 # slices of one fused projection
        s["start"], s["nq"] = None, nk if case["ragged"] else None
        qkv = rnd(b, (h + 2 * hk) * d, tk).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :h * d], qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
    s["nk"] = nk if case["ragged"] or case["last"] else None
    s["bias"] = rnd(h, case["buckets"])
    s["map"] = _bucket_map(case).to(dev)
    if case["op"] == "attend_grad":
        s["dout"] = rnd(b, h * d, tq).to(dt)
        s["out"], s["lse"] = _attend(s)
    if own:
        from vits_amd import attention
        s["buckets"] = attention.RelativeBuckets(case["buckets"], case["distance"], bidirectional=not case["causal"])
        s["buckets"].table(dev)
    return s


def _bucket_map(case):
    """Bucket of every offset key - query from -distance to distance (further ones as at the ends):
    half of the buckets for either sign (all for a causal case, where the keys ahead share bucket 0),
    of these half for one distance each and half for ranges that grow in proportion.  Whole-number
    arithmetic, so that no border depends on a rounding."""
    nb, far = case["buckets"], case["distance"]
    if not case["causal"]:
        nb //= 2
    exact_n = nb // 2
    m = nb - exact_n

    def bucket(n):
        if n < exact_n:
            return n
        k = 0
        while k + 1 < m and n ** m * exact_n ** (k + 1) >= far ** (k + 1) * exact_n ** m:
            k += 1
        return exact_n + k

    return torch.tensor([(nb if o > 0 and not case["causal"] else 0)
                         + (bucket(abs(o)) if o < 0 or not case["causal"] else 0) for o in range(-far, far + 1)])


# ---- the operators --------------------------------------------------------------------------------

def run(s):
    return _OPS[s["case"]["op"]](s) if not own else _OWN[s["case"]["op"]](s)


def _geometry(s):
    """Offsets key - query [1 or B, Tq, Tk] and which pairs are allowed (broadcasts to [B, Tq, Tk])."""
    c = s["case"]
    dev, tq, tk = s["q"].device, c["queries"], c["keys"]
    j = torch.arange(tk, device=dev).view(1, 1, tk)
    i = torch.arange(tq, device=dev).view(1, tq, 1)
    off = j - (i if s["start"] is None else i + s["start"].view(-1, 1, 1))
    ok = torch.ones(1, 1, 1, dtype=torch.bool, device=dev)
    if s["nk"] is not None:
        ok = ok & (j < s["nk"].view(-1, 1, 1))
    if s["nq"] is not None:
        ok = ok & (i < s["nq"].view(-1, 1, 1))
    if c["causal"]:
        ok = ok & (off <= 0)
    return off, ok


def _split_heads(x, n, group=1):
    b, hd, t = x.shape
    x = x.float().view(b, n, hd // n, t)
    return x.repeat_interleave(group, dim=1) if group > 1 else x


def _scores(s):
    """Logits [B, H, Tq, Tk] in 32 bits, -inf where a pair is not allowed, with q and k by heads."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    q, k = _split_heads(s["q"], c["heads"]), _split_heads(s["k"], c["kv_heads"], group)
    off, ok = _geometry(s)
    where = s["map"][off.clamp(-c["distance"], c["distance"]) + c["distance"]]
    bias = s["bias"][:, where].transpose(0, 1)             # [1 or B, H, Tq, Tk]
    a = torch.matmul(q.transpose(2, 3), k) * (1 / math.sqrt(c["dim"]))
    a = (a + bias).masked_fill_(~ok.unsqueeze(1), -math.inf)
    return a, q, k, off


def _attend(s):
    c = s["case"]
    a, _, _, _ = _scores(s)
    top = a.amax(-1, keepdim=True)
    p = torch.exp(a - top.masked_fill(top == -math.inf, 0))
    del a
    total = p.sum(-1, keepdim=True)
    v = _split_heads(s["v"], c["kv_heads"], c["heads"] // c["kv_heads"])
    o = torch.matmul(p, v.transpose(2, 3).contiguous()) / total.masked_fill(total == 0, 1)
    lse = (top + torch.log(total)).squeeze(-1)
    b, h, tq, d = o.shape
    return o.transpose(2, 3).reshape(b, h * d, tq).to(s["q"].dtype), lse


def _attend_grad(s):
    c = s["case"]
    b, h, hk, d, tq, tk = (c[n] for n in ("batch", "heads", "kv_heads", "dim", "queries", "keys"))
    a, q, k, off = _scores(s)
    lse = s["lse"].unsqueeze(-1)
    p = torch.exp(a - lse.masked_fill(lse == -math.inf, 0))
    del a
    do, o = _split_heads(s["dout"], h), _split_heads(s["out"], h)
    v = _split_heads(s["v"], hk, h // hk)
    dv = torch.matmul(do, p)                                                        # [B, H, D, Tk]
    ds = torch.matmul(do.transpose(2, 3), v).sub_((do * o).sum(2).unsqueeze(-1)).mul_(p)
    del p
    scale = 1 / math.sqrt(d)
    dq = torch.matmul(k, ds.transpose(2, 3).contiguous()) * scale                   # [B, H, D, Tq]
    dk = torch.matmul(q, ds) * scale
    # sums along the diagonals key - query = const: rows in reverse order, each one place further right
    skew = torch.nn.functional.pad(ds.flip(2), (0, tq)).flatten(2)[..., :tq * (tq + tk) - tq]
    diag = skew.view(b, h, tq, tq + tk - 1).sum(2, dtype=torch.float64)              # offset index - (tq - 1)
    first = off[:, tq - 1, 0].view(-1, 1) + torch.arange(tq + tk - 1, device=off.device)
    where = s["map"][first.clamp(-c["distance"], c["distance"]) + c["distance"]].expand(b, -1)
    one_hot = (where.unsqueeze(-1) == torch.arange(c["buckets"], device=off.device)).double()
    dbias = torch.matmul(diag, one_hot).sum(0).float()
    dt = s["q"].dtype
    dk, dv = (g.view(b, hk, h // hk, d, tk).sum(2).view(b, hk * d, tk).to(dt) for g in (dk, dv))
    return dq.reshape(b, h * d, tq).to(dt), dk, dv, dbias


def _normed(x, kind):
    """x over its root mean square (or its deviation, without its mean) along the channels, and that factor."""
    x = x.float()
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5)
    return x * r, r


def _norm_back(dy, xhat, r, kind):
    g = dy - xhat * (dy * xhat).mean(1, keepdim=True)
    if kind == "layer":
        g = g - dy.mean(1, keepdim=True)
    return g * r


def _col(p):
    return p.view(1, -1, 1)


def _inside(s, t):
    if s["lengths"] is None:
        return None
    return (torch.arange(t, device=s["lengths"].device) < s["lengths"].view(-1, 1)).unsqueeze(1)


def _block_norm(s):
    kind = s["case"]["norm"]
    xhat, _ = _normed(s["y"], kind)
    z = xhat * _col(s["post"][0])
    if s["post"][1] is not None:
        z = z + _col(s["post"][1])
    h = s["x"].float() + _col(s["scale"]) * s["gate"].float() * z
    hhat, _ = _normed(h, kind)
    n = hhat * _col(s["pre"][0])
    if s["pre"][1] is not None:
        n = n + _col(s["pre"][1])
    ok = _inside(s, h.shape[2])
    if ok is not None:
        h, n = h.masked_fill(~ok, 0), n.masked_fill(~ok, 0)
    dt = s["x"].dtype
    return h.to(dt), n.to(dt)


def _block_norm_grad(s):
    kind = s["case"]["norm"]
    ok = _inside(s, s["h"].shape[2])
    dh, dn = s["dh"].float(), s["dn"].float()
    if ok is not None:
        dh, dn = dh.masked_fill(~ok, 0), dn.masked_fill(~ok, 0)
    over = lambda x: x.sum((0, 2))  # noqa: E731
    hhat, hr = _normed(s["h"], kind)
    dh = dh + _norm_back(dn * _col(s["pre"][0]), hhat, hr, kind)
    yhat, yr = _normed(s["y"], kind)
    z = yhat * _col(s["post"][0])
    if s["post"][1] is not None:
        z = z + _col(s["post"][1])
    gate = s["gate"].float()
    dz = dh * _col(s["scale"]) * gate
    dgate = dh * _col(s["scale"]) * z
    if gate.shape[2] == 1:
        dgate = dgate.sum(2, keepdim=True)
    dy = _norm_back(dz * _col(s["post"][0]), yhat, yr, kind)
    dt = s["h"].dtype
    grads = {"dx": dh.to(dt), "dy": dy.to(dt), "dgate": dgate.to(dt), "dscale": over(dh * gate * z),
             "dpost": over(dz * yhat), "dpre": over(dn * hhat)}
    if kind == "layer":
        grads |= {"dpost_bias": over(dz), "dpre_bias": over(dn)}
    return grads


def _own_attend(s):
    from vits_amd import attention
    c = s["case"]
    return attention.bucket_attention(s["q"], s["k"], s["v"], s["bias"], s["buckets"], heads=c["heads"],
                                      kv_heads=c["kv_heads"], key_lengths=s["nk"], query_lengths=s["nq"],
                                      query_start=s["start"], causal=c["causal"], return_lse=True)


def _own_attend_grad(s):
    from vits_amd import attention
    c = s["case"]
    return attention.bucket_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["bias"],
                                               s["buckets"], heads=c["heads"], kv_heads=c["kv_heads"],
                                               key_lengths=s["nk"], query_lengths=s["nq"], query_start=s["start"],
                                               causal=c["causal"])


def _own_norm(s):
    from vits_amd import block_norm
    return block_norm.block_norm(s["x"], s["y"], post=s["post"], gate=s["gate"], scale=s["scale"], pre=s["pre"],
                                 norm=s["case"]["norm"], lengths=s["lengths"])


def _own_norm_grad(s):
    from vits_amd import block_norm
    g = block_norm.block_norm_backward(s["dh"], s["dn"], s["h"], s["y"], post=s["post"], gate=s["gate"],
                                       scale=s["scale"], pre=s["pre"], norm=s["case"]["norm"], lengths=s["lengths"])
    r = {"dx": g.x, "dy": g.y, "dgate": g.gate, "dscale": g.scale, "dpost": g.post[0], "dpre": g.pre[0]}
    if s["case"]["norm"] == "layer":
        r |= {"dpost_bias": g.post[1], "dpre_bias": g.pre[1]}
    return r


_OPS = {"attend": _attend, "attend_grad": _attend_grad, "norm": _block_norm, "norm_grad": _block_norm_grad}
_OWN = {"attend": _own_attend, "attend_grad": _own_attend_grad, "norm": _own_norm, "norm_grad": _own_norm_grad}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    b = case["batch"]
    if case["op"] in ("norm", "norm_grad"):
        c, t = case["channels"], case["length"]
        n, full = sum(_lengths(case, t)) * c, b * c * t
        gate = n if case["gate"] == "full" else b * c
        if case["op"] == "norm":                            # x, y, gate in; h, n out
            return {"bytes": size * (2 * n + gate + 2 * full) + 20 * c, "flops": 20 * n}
        dgate = full if case["gate"] == "full" else b * c   # dh, dn, h, y, gate in; dx, dy, dgate out
        return {"bytes": size * (4 * n + gate + 2 * full + dgate) + 40 * c, "flops": 40 * n}
    h, hk, d, tq, tk = (case[n] for n in ("heads", "kv_heads", "dim", "queries", "keys"))
    pairs, nq_all, nk_all = 0, 0, 0
    for nk in _lengths(case, tk):
        nq, start = (tq, nk - tq) if case["last"] else (nk, 0)
        nq_all, nk_all = nq_all + nq, nk_all + nk
        if case["causal"]:
            pairs += sum(max(0, min(nk, start + i + 1)) for i in range(nq))
        else:
            pairs += nq * nk
    qb, kb, lse = size * h * d * nq_all, size * hk * d * nk_all, 4 * h * nq_all
    if case["op"] == "attend":
        return {"bytes": 2 * qb + 2 * kb + lse, "flops": 4 * d * h * pairs}
    return {"bytes": 4 * qb + 4 * kb + lse, "flops": 10 * d * h * pairs}


# ---- the definition in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"] == "norm_grad":
        return _exact_norm_grad(case, s)
    return _exact_attend(case, s)


def _exact_attend(case, s):
    """One item and head at a time, rows in blocks."""
    b, h, hk, d, tq, tk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "queries", "keys"))
    if b * h * tq * tk > 4e9:
        return None
    grad = case["op"] == "attend_grad"
    dev = s["q"].device
    heads = lambda x, n: x.double().reshape(b, n, d, -1)  # noqa: E731
    q, k, v = heads(s["q"], h), heads(s["k"], hk), heads(s["v"], hk)
    out = torch.zeros(b, h, d, tq, dtype=torch.float64, device=dev)
    lse = torch.full((b, h, tq), -math.inf, dtype=torch.float64, device=dev)
    if grad:
        do, o, left = heads(s["dout"], h), heads(s["out"], h), s["lse"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dbias = torch.zeros(h, case["buckets"], dtype=torch.float64, device=dev)
    for bi in range(b):
        n_k = tk if s["nk"] is None else int(s["nk"][bi])
        n_q = tq if s["nq"] is None else int(s["nq"][bi])
        start = 0 if s["start"] is None else int(s["start"][bi])
        for at in range(0, n_q, 2048):
            rows = torch.arange(at, min(n_q, at + 2048), device=dev)
            rel = torch.arange(n_k, device=dev)[None, :] - (rows[:, None] + start)
            bucket = s["map"][rel.clamp(min=-case["distance"], max=case["distance"]) + case["distance"]]
            for hi in range(h):
                g = hi * hk // h
                logit = (q[bi, hi][:, rows].T @ k[bi, g][:, :n_k]) / math.sqrt(d) + s["bias"].double()[hi][bucket]
                if case["causal"]:
                    logit = logit.where(rel <= 0, torch.full((), -math.inf, dtype=torch.float64, device=dev))
                if not grad:
                    lse[bi, hi, rows] = torch.logsumexp(logit, 1)
                    w = torch.softmax(logit, 1).nan_to_num(0.0) if n_k else logit
                    out[bi, hi][:, rows] = v[bi, g][:, :n_k] @ w.T
                    continue
                w = torch.exp(logit - left[bi, hi, rows][:, None]) * (left[bi, hi, rows][:, None] > -math.inf)
                dor = do[bi, hi][:, rows]
                dlogit = w * (dor.T @ v[bi, g][:, :n_k] - (dor * o[bi, hi][:, rows]).sum(0)[:, None])
                dq[bi, hi][:, rows] = k[bi, g][:, :n_k] @ dlogit.T / math.sqrt(d)
                dk[bi, g][:, :n_k] += q[bi, hi][:, rows] @ dlogit / math.sqrt(d)
                dv[bi, g][:, :n_k] += dor @ w
                for c in range(case["buckets"]):
                    dbias[hi, c] += (dlogit * (bucket == c)).sum()
    if not grad:
        return out.reshape(b, h * d, tq), lse
    return dq.reshape(b, h * d, tq), dk.reshape(b, hk * d, tk), dv.reshape(b, hk * d, tk), dbias


def _exact_parts(v, norm):
    v = v.double()
    mean = v.mean(1, keepdim=True) if norm == "layer" else torch.zeros_like(v[:, :1])
    dev2 = ((v - mean) ** 2).mean(1, keepdim=True)
    return (v - mean) / torch.sqrt(dev2 + 1e-5), torch.sqrt(dev2 + 1e-5)


def _exact_affine(unit, p):
    z = unit * p[0].double()[None, :, None]
    return z if p[1] is None else z + p[1].double()[None, :, None]


def _exact_keep(s, x):
    if s["lengths"] is not None:
        for i, n in enumerate(s["lengths"].tolist()):
            x[i, :, n:] = 0
    return x


def _exact_norm(case, s):
    z = _exact_affine(_exact_parts(s["y"], case["norm"])[0], s["post"])
    h = s["x"].double() + s["scale"].double()[None, :, None] * s["gate"].double() * z
    n = _exact_affine(_exact_parts(h, case["norm"])[0], s["pre"])
    return _exact_keep(s, h), _exact_keep(s, n)


def _exact_norm_grad(case, s):
    """d unit / d v = (1 - 1/C - unit unit^T / C) / dev, without the 1/C where no mean is taken."""
    layer = case["norm"] == "layer"

    def through(g, unit, dev):
        c = unit.shape[1]
        back = g - unit * ((g * unit).sum(1, keepdim=True) / c)
        return (back - g.sum(1, keepdim=True) / c if layer else back) / dev

    dh, dn = _exact_keep(s, s["dh"].double()), _exact_keep(s, s["dn"].double())
    unit_h, dev_h = _exact_parts(s["h"], case["norm"])
    dx = dh + through(dn * s["pre"][0].double()[None, :, None], unit_h, dev_h)
    unit_y, dev_y = _exact_parts(s["y"], case["norm"])
    z, gate, scale = _exact_affine(unit_y, s["post"]), s["gate"].double(), s["scale"].double()[None, :, None]
    dz = dx * gate * scale
    dgate = dx * z * scale
    if case["gate"] == "item":
        dgate = dgate.sum(2, keepdim=True)
    r = {"dx": dx, "dy": through(dz * s["post"][0].double()[None, :, None], unit_y, dev_y), "dgate": dgate,
         "dscale": (dx * gate * z).sum(2).sum(0), "dpost": (dz * unit_y).sum(2).sum(0),
         "dpre": (dn * unit_h).sum(2).sum(0)}
    if layer:
        r |= {"dpost_bias": dz.sum(2).sum(0), "dpre_bias": dn.sum(2).sum(0)}
    return r
