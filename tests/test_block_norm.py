"""The norms around a block, its gate, scale and residual sum, forward and backward, against the definition in 64 bits.

Tolerances are bounds on the rounding errors per element, with u = 2^-24 (half a step of fp32) and the half step of the
stored type: a sum over n terms is off by at most n u of the sum of their magnitudes (the kernels add in trees, so this
is generous), each elementary operation by u of its result, a stored result by its type's half step."""
import ctypes as C
import math

import pytest
import torch

from vits_amd import native
from vits_amd.block_norm import block_norm, block_norm_backward

gpu = pytest.mark.gpu
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Norm:
    """unit = (v - mean) / dev of a [B, C, T] value that is itself only known within `e`, with the bound of its error."""

    def __init__(self, v, kind, eps, e=0.0):
        n = v.shape[1]
        self.layer, self.n = kind == "layer", n
        mean = v.mean(1, keepdim=True) if self.layer else torch.zeros_like(v[:, :1])
        self.dev = ((v - mean).square().mean(1, keepdim=True) + eps).sqrt()
        self.unit = (v - mean) / self.dev
        e = e + torch.zeros_like(v)
        e_mean = e.mean(1, keepdim=True) + (n + 2) * U * v.abs().mean(1, keepdim=True) if self.layer else 0.0
        e_c = e + e_mean + U * (v - mean).abs()
        # relative error of dev: half of that of its square
        rel = ((e_c * (v - mean).abs()).mean(1, keepdim=True) + e_c.square().mean(1, keepdim=True)) / self.dev.square() + (n + 8) * U
        self.rel = rel
        self.e = e_c / self.dev * (1 + rel) + self.unit.abs() * (rel + 4 * U)

    def back(self, g, e_g):
        """Gradient through the norm and its bound."""
        n = self.n
        u, eu = self.unit, self.e
        m1 = g.mean(1, keepdim=True) if self.layer else torch.zeros_like(g[:, :1])
        m2 = (g * u).mean(1, keepdim=True)
        e1 = e_g.mean(1, keepdim=True) + (n + 2) * U * g.abs().mean(1, keepdim=True) if self.layer else 0.0
        e2 = (e_g * u.abs() + g.abs() * eu + e_g * eu).mean(1, keepdim=True) + (n + 3) * U * (g * u).abs().mean(1, keepdim=True)
        r = (g - m1 - u * m2) / self.dev
        size = (g.abs() + m1.abs() + (u * m2).abs()) / self.dev
        e = (e_g + e1 + u.abs() * e2 + eu * (m2.abs() + e2)) / self.dev * (1 + self.rel) + size * (self.rel + 8 * U)
        return r, e


def reference(x, y, gate, scale, post, pre, kind, eps, lengths, dh=None, dn=None, h_given=None):
    """{name: (value, bound)} in 64 bits on the CPU."""
    dt = x.dtype if x is not None else h_given.dtype
    cpu = lambda t: None if t is None else t.detach().cpu().double()
    col = lambda t: t.view(1, -1, 1)
    like = x if x is not None else h_given
    B, Cn, T = like.shape
    ok = torch.ones(B, 1, T, dtype=torch.bool) if lengths is None else (torch.arange(T) < lengths.cpu().clamp(0, T).view(-1, 1)).unsqueeze(1)
    clean = lambda t: None if t is None else torch.where(ok if t.shape[2] == T else torch.ones_like(ok[:, :, :1]), cpu(t), torch.zeros((), dtype=torch.float64))
    x, y, dh, dn, h_given = clean(x), clean(y), clean(dh), clean(dn), clean(h_given)
    if gate is not None:
        per_item = gate.shape[2] == 1 and T != 1
        gate = cpu(gate) if per_item else clean(gate)
    store = lambda v, e, d: (v, e + half_step(d) * (v.abs() + e) + 1e-30)
    keep = lambda v: torch.where(ok, v, torch.zeros((), dtype=v.dtype))
    res = {}
    ny = None
    if y is not None:
        if post is not None:
            ny = Norm(y, kind, eps)
            w, b = col(cpu(post[0])), col(cpu(post[1])) if post[1] is not None else torch.zeros(1, 1, 1, dtype=torch.float64)
            z = ny.unit * w + b
            ez = ny.e * w.abs() + 2 * U * (ny.unit * w).abs() + U * z.abs()
        else:
            z, ez = y, torch.zeros_like(y)
        s = col(cpu(scale)) if scale is not None else torch.ones(1, 1, 1, dtype=torch.float64)
        g = gate if gate is not None else torch.ones(1, 1, 1, dtype=torch.float64)
    if dh is None and dn is None:
        h, eh = x, torch.zeros_like(x)
        if y is not None:
            h = x + s * g * z
            eh = (s * g).abs() * ez + 3 * U * (s * g * z).abs() + U * h.abs()
            res["h"] = store(keep(h), keep(eh), dt)
        if pre is not None:
            nh = Norm(h, kind, eps, eh)
            w, b = col(cpu(pre[0])), col(cpu(pre[1])) if pre[1] is not None else torch.zeros(1, 1, 1, dtype=torch.float64)
            n = nh.unit * w + b
            res["n"] = store(keep(n), keep(nh.e * w.abs() + 2 * U * (nh.unit * w).abs() + U * n.abs()), dt)
        return res
    cols = B * T + 8
    total = lambda v, e: ((v.sum((0, 2))), (e.sum((0, 2)) + cols * U * v.abs().sum((0, 2))))
    store_sum = lambda v, e: store(*total(keep(v), keep(e)), torch.float32)
    gr, eg = (dh, torch.zeros_like(dh)) if dh is not None else (torch.zeros(B, Cn, T, dtype=torch.float64),) * 2
    if dn is not None:
        nh = Norm(h_given, kind, eps)
        w = col(cpu(pre[0]))
        back, eb = nh.back(dn * w, U * (dn * w).abs())
        res["dw_pre"] = store_sum(dn * nh.unit, dn.abs() * nh.e + 2 * U * (dn * nh.unit).abs())
        res["db_pre"] = store_sum(dn, torch.zeros_like(dn))
        gr, eg = gr + back, eb + U * (gr + back).abs()
    res["dx"] = store(keep(gr), keep(eg), dt)
    if y is None:
        return res
    dgate, e = gr * s * z, (s * z).abs() * eg + (gr * s).abs() * ez + eg * s.abs() * ez + 3 * U * (gr * s * z).abs()
    if gate is not None:
        if per_item:
            v, b = keep(dgate), keep(e)
            res["dgate"] = store(v.sum(2, keepdim=True), b.sum(2, keepdim=True) + (T + 8) * U * v.abs().sum(2, keepdim=True), dt)
        else:
            res["dgate"] = store(keep(dgate), keep(e), dt)
    dsv = gr * g * z
    res["dscale"] = store_sum(dsv, (g * z).abs() * eg + (gr * g).abs() * ez + eg * g.abs() * ez + 3 * U * dsv.abs())
    dz, edz = gr * s * g, (s * g).abs() * eg + 3 * U * (gr * s * g).abs()
    if ny is not None:
        res["dw_post"] = store_sum(dz * ny.unit, edz * ny.unit.abs() + dz.abs() * ny.e + edz * ny.e + 2 * U * (dz * ny.unit).abs())
        res["db_post"] = store_sum(dz, edz)
        w = col(cpu(post[0]))
        dy, edy = ny.back(dz * w, edz * w.abs() + U * (dz * w).abs())
    else:
        dy, edy = dz, edz
    res["dy"] = store(keep(dy), keep(edy), dt)
    return res


def assert_within(name, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), name
    off = (got - value).abs() - bound
    if off.numel():
        i = off.argmax()
        assert off.max() <= 0, (name, float(got.flatten()[i]), float(value.flatten()[i]), float(bound.flatten()[i]))


def inputs(dtype, B, Cn, T, *, gate="full", scale=True, post=True, pre=True, bias=True, y=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    big = lambda: rnd(B, Cn, T).to(dtype).cuda()
    d = dict(x=big(), y=(rnd(B, Cn, T) * 1.5 + 0.3).to(dtype).cuda() if y else None)
    d["gate"] = None if gate is None or not y else (rnd(B, Cn, T if gate == "full" else 1) * 0.5 + 1).to(dtype).cuda()
    d["scale"] = (rnd(Cn) * 0.2 + 0.5).cuda() if scale and y else None
    pair = lambda: ((rnd(Cn) * 0.3 + 1).cuda(), (rnd(Cn) * 0.2).cuda() if bias else None)
    d["post"] = pair() if post and y else None
    d["pre"] = pair() if pre else None
    return d, big(), big()


# B, C, T, options
CASES = [
    (1, 192, 43, dict()),                                        # one sentence of the text encoder
    (1, 1, 1, dict()),
    (2, 3, 5, dict(gate="item")),
    (3, 192, 131, dict(gate="item", lengths=[131, 0, 57])),
    (2, 257, 64, dict(norm="rms", bias=False)),
    (2, 1024, 33, dict(norm="rms", gate="item", lengths=[33, 8])),
    (1, 2048, 19, dict()),
    (1, 4096, 9, dict(gate=None, scale=False)),
    (2, 100, 77, dict(post=False)),
    (2, 100, 77, dict(pre=False, gate=None)),
    (2, 100, 77, dict(post=False, gate=None, scale=False)),      # a plain residual sum and norm
    (2, 130, 40, dict(y=False, lengths=[40, 21])),               # the first norm of a stack
    (40, 192, 300, dict(lengths=[300 - 7 * i for i in range(40)])),
    (24, 640, 161, dict(norm="rms", gate="item")),
    (2, 513, 2500, dict()),
]
IDS = [f"B{b}C{c}T{t}-" + "-".join(f"{k}" for k in o) for b, c, t, o in CASES]


def split_options(o):
    o = dict(o)
    lengths = o.pop("lengths", None)
    return o.pop("norm", "layer"), None if lengths is None else torch.tensor(lengths, device="cuda"), o


def grads_dict(g):
    d = {"dx": g.x, "dy": g.y, "dgate": g.gate, "dscale": g.scale}
    for name, pair in (("post", g.post), ("pre", g.pre)):
        if pair is not None:
            d["dw_" + name], d["db_" + name] = pair
    return {k: v for k, v in d.items() if v is not None}


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,Cn,T,opts", CASES, ids=IDS)
def test_forward_and_backward(B, Cn, T, opts, dtype):
    norm, lengths, o = split_options(opts)
    d, dh, dn = inputs(dtype, B, Cn, T, **o)
    h, n = block_norm(**d, norm=norm, lengths=lengths)
    ref = reference(d["x"], d["y"], d["gate"], d["scale"], d["post"], d["pre"], norm, 1e-5, lengths)
    if d["y"] is not None:
        assert_within("h", h, ref["h"])
    if d["pre"] is not None:
        assert_within("n", n, ref["n"])
    else:
        assert n is None
    keep = {k: v for k, v in d.items() if k not in ("x", "y")}
    for a, b in ((dh, dn), (None, dn), (dh, None)):
        if b is not None and d["pre"] is None:
            b = None
            if a is None:
                continue
        grads = grads_dict(block_norm_backward(a, b, h, d["y"], **keep, norm=norm, lengths=lengths))
        ref = reference(None, d["y"], d["gate"], d["scale"], d["post"], d["pre"], norm, 1e-5, lengths, a, b, h)
        for name, g in grads.items():
            assert_within(name, g, ref[name])
        again = grads_dict(block_norm_backward(a, b, h, d["y"], **keep, norm=norm, lengths=lengths))
        assert all(torch.equal(grads[k], again[k]) for k in grads), "the same inputs give the same bits"


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_columns_far_from_zero_and_constant_ones(dtype, norm):
    """A mean a thousand times the spread, and columns without any spread."""
    d, dh, dn = inputs(dtype, 2, 192, 50)
    d["y"] = (d["y"].float() + 1000).to(dtype)
    d["y"][:, :, 7] = 3.0
    d["x"][:, :, 9] = 0.0
    d["gate"][:, :, 9] = 0.0
    h, n = block_norm(**d, norm=norm)
    ref = reference(d["x"], d["y"], d["gate"], d["scale"], d["post"], d["pre"], norm, 1e-5, None)
    assert_within("h", h, ref["h"])
    assert_within("n", n, ref["n"])
    keep = {k: v for k, v in d.items() if k not in ("x", "y")}
    ref = reference(None, d["y"], d["gate"], d["scale"], d["post"], d["pre"], norm, 1e-5, None, dh, dn, h)
    for name, g in grads_dict(block_norm_backward(dh, dn, h, d["y"], **keep, norm=norm)).items():
        assert_within(name, g, ref[name])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_padding_may_hold_anything(dtype):
    lengths = torch.tensor([60, 0, 23], device="cuda")
    d, dh, dn = inputs(dtype, 3, 96, 60)
    pad = torch.arange(60, device="cuda").view(1, 1, -1) >= lengths.view(-1, 1, 1)
    run = lambda d, dh, dn, h=None: (lambda hn: (*hn, grads_dict(block_norm_backward(
        dh, dn, hn[0] if h is None else h, d["y"], gate=d["gate"], scale=d["scale"], post=d["post"], pre=d["pre"], lengths=lengths))))(
        block_norm(**d, lengths=lengths))
    h, n, g = run(d, dh, dn)
    assert not h.masked_select(pad).any() and not n.masked_select(pad).any()
    for val in (math.nan, math.inf):
        dirty = lambda t: t.masked_fill(pad, val)
        d2 = d | {k: dirty(d[k]) for k in ("x", "y", "gate")}
        h2, n2, g2 = run(d2, dirty(dh), dirty(dn), dirty(h))
        assert torch.equal(h, h2) and torch.equal(n, n2) and all(torch.equal(g[k], g2[k]) for k in g)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_views_and_surroundings(dtype):
    """Inputs cut out of larger tensors at odd places give the same bits, outputs in views leave the rest alone."""
    d, dh, dn = inputs(dtype, 2, 70, 91)

    def cut(t):
        big = torch.full((t.shape[0] + 1, t.shape[1] + 5, t.shape[2] + 6), 7.0, device="cuda", dtype=t.dtype)
        v = big[1:, 2:2 + t.shape[1], 3:3 + t.shape[2]]
        v.copy_(t)
        return big, v

    want_h, want_n = block_norm(**d)
    v = d | {k: cut(d[k])[1] for k in ("x", "y", "gate")}
    h, n = block_norm(**v)
    assert torch.equal(h, want_h) and torch.equal(n, want_n)
    rooms = [cut(torch.zeros_like(d["x"])) for _ in range(5)]
    p = dict(gate=v["gate"], scale=d["scale"], post=d["post"], pre=d["pre"])
    native.block_norm(v["x"], v["y"], rooms[0][1], rooms[1][1], **p)
    keep = {k: t for k, t in d.items() if k not in ("x", "y")}
    want = block_norm_backward(dh, dn, want_h, d["y"], **keep)
    native.block_norm_backward(cut(dh)[1], cut(dn)[1], rooms[0][1], v["y"], rooms[2][1], rooms[3][1], dgate=rooms[4][1], **p)
    for (big, view), w in zip(rooms, (want_h, want_n, want.x, want.y, want.gate)):
        assert torch.equal(view, w)
        view.fill_(7.0)
        assert (big == 7.0).all()


@gpu
def test_autograd_and_differences():
    lengths = torch.tensor([37, 20], device="cuda")
    d, dh, dn = inputs(torch.float32, 2, 48, 37, gate="item")
    flat = [d["x"], d["y"], d["gate"], d["scale"], *d["post"], *d["pre"]]
    call = lambda x, y, gate, scale, wp, bp, wn, bn: block_norm(x, y, post=(wp, bp), gate=gate, scale=scale, pre=(wn, bn), lengths=lengths)
    with torch.enable_grad():
        leaves = [t.clone().requires_grad_() for t in flat]
        h, n = call(*leaves)
        got = torch.autograd.grad((h, n), leaves, (dh, dn))
        only_n = torch.autograd.grad(call(*leaves)[1].sum(), leaves)           # an expanded gradient, none for h
        only_h = torch.autograd.grad(call(*leaves)[0], leaves[:6], dh)
    h, n = call(*flat)
    opts = {k: v for k, v in d.items() if k not in ("x", "y")} | dict(lengths=lengths)
    unpacked = lambda g: (g.x, g.y, g.gate, g.scale, *(g.post or ()), *(g.pre or ()))
    assert all(torch.equal(a, b) for a, b in zip(got, unpacked(block_norm_backward(dh, dn, h, d["y"], **opts))))
    assert all(torch.equal(a, b) for a, b in zip(only_n, unpacked(block_norm_backward(None, torch.ones_like(dn), h, d["y"], **opts))))
    assert all(torch.equal(a, b) for a, b in zip(only_h, unpacked(block_norm_backward(dh, None, h, d["y"], **opts))))
    # the derivative of the 64-bit definition along random directions
    at = [t.cpu().double() for t in flat]

    def f(x, y, gate, scale, wp, bp, wn, bn):
        r = reference(x, y, gate, scale, (wp, bp), (wn, bn), "layer", 1e-5, lengths)
        return float((r["h"][0] * dh.cpu()).sum() + (r["n"][0] * dn.cpu()).sum())

    ref = reference(None, d["y"], d["gate"], d["scale"], d["post"], d["pre"], "layer", 1e-5, lengths, dh, dn, h)
    names = ("dx", "dy", "dgate", "dscale", "dw_post", "db_post", "dw_pre", "db_pre")
    g = torch.Generator().manual_seed(5)
    inside = (torch.arange(37) < lengths.cpu().view(-1, 1)).unsqueeze(1)
    for i, name in enumerate(names):
        step = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        if step.shape == (2, 48, 37):
            step = step * inside
        eps = 1e-5
        moved = [[t + sign * eps * step if j == i else t for j, t in enumerate(at)] for sign in (1, -1)]
        diff = (f(*moved[0]) - f(*moved[1])) / (2 * eps)
        along = float((got[i].cpu().double() * step).sum())
        # h as stored differs from the exact one by half an fp32 step: an unit's relative change times the sums' size
        slack = 1e-6 * float((ref[name][0].abs() * step.abs()).sum()) + 1e-6 * max(1.0, abs(diff))
        assert abs(diff - along) <= float((ref[name][1] * step.abs()).sum()) + slack, name


@gpu
def test_empty_sizes_graphs_and_streams():
    z = torch.zeros(2, 8, 0, device="cuda")
    w = torch.ones(8, device="cuda")
    h, n = block_norm(z, z, post=(w, w), pre=(w, w))
    assert h.shape == n.shape == z.shape
    g = block_norm_backward(z, z, z, z, post=(w, w), pre=(w, w), scale=w)
    assert not g.post[0].any() and not g.pre[1].any() and not g.scale.any()
    sets = [inputs(torch.bfloat16, b, c, t, gate="item", seed=t) for b, c, t in ((1, 192, 1), (2, 320, 77), (3, 64, 500))]

    def step(d, dh, dn):
        h, n = block_norm(**d)
        g = block_norm_backward(dh, dn, h, d["y"], **{k: v for k, v in d.items() if k not in ("x", "y")})
        return (h, n, *grads_dict(g).values())

    want = [step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for x, y in zip(got, want) for p, q in zip(x, y))
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(*s)
        graphs.append((gr, res))
    for _ in range(3):
        for (gr, res), s, want_s in zip(graphs, sets, want):
            for t in res:
                t.fill_(3.0)
            gr.replay()
            step(*sets[1])
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(res, want_s))


@gpu
def test_refusals():
    d, dh, dn = inputs(torch.float32, 2, 16, 12)
    bad = [dict(x=d["x"].half()), dict(x=d["x"][0]), dict(y=d["y"].bfloat16()), dict(y=d["y"][:, :, :5]), dict(gate=d["gate"][:, :8]),
           dict(gate=d["gate"][:, :, :5]), dict(scale=d["scale"][:3]), dict(scale=d["scale"].double()), dict(post=(None, d["scale"])),
           dict(pre=(d["scale"].bfloat16(), None)), dict(norm="batch"), dict(eps=0.0), dict(lengths=torch.tensor([1, 2])),
           dict(lengths=torch.tensor([1], device="cuda")), dict(y=None), dict(x=d["x"].transpose(1, 2).contiguous().transpose(1, 2))]
    for change in bad:
        with pytest.raises(ValueError):
            block_norm(**(d | change))
    with pytest.raises(ValueError):
        block_norm(d["x"])
    keep = {k: v for k, v in d.items() if k not in ("x", "y")}
    for args in ((None, None, d["x"]), (dh[:1], dn, d["x"]), (dh.bfloat16(), dn, d["x"]), (dh, dn[:, :, :3], d["x"])):
        with pytest.raises(ValueError):
            block_norm_backward(*args, d["y"], **keep)
    with pytest.raises(ValueError):
        block_norm_backward(dh, dn, d["x"], d["y"], **(keep | dict(pre=None)))
    wide = torch.zeros(1, 4097, 2, device="cuda")
    with pytest.raises(ValueError):
        block_norm(wide, wide)


@gpu
def test_capture_under_autograd_is_refused():
    d, _, _ = inputs(torch.float32, 1, 16, 8)
    block_norm(**d)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    keep = torch.zeros(1, device="cuda")
    with torch.enable_grad(), torch.cuda.graph(gr):
        keep.add_(1)
        with pytest.raises(native.NativeError, match="captured"):
            block_norm(d["x"].requires_grad_(), d["y"], pre=d["pre"])


# ---- on the CPU ------------------------------------------------------------------------------------

def _args(**kw):
    a = native.BlockNormArgs()
    for n in ("x", "y", "gate", "h", "n", "dh", "dn", "dx", "dy", "dgate"):
        setattr(a, n, 4096), setattr(a, n + "_bstride", 6400), setattr(a, n + "_cstride", 100)
    for n in ("scale", "w_post", "b_post", "w_pre", "b_pre", "dscale", "dw_post", "db_post", "dw_pre", "db_pre"):
        setattr(a, n, 4096)
    a.batch, a.channels, a.length, a.eps = 2, 64, 100, 1e-5
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad,code", [
    (dict(batch=-1), -1), (dict(channels=0), -1), (dict(length=-1), -1), (dict(dtype=2), -2), (dict(norm=2), -1),
    (dict(channels=4097), -2), (dict(eps=0.0), -1), (dict(eps=float("nan")), -1), (dict(y=0), -1), (dict(w_post=0), -1),
    (dict(w_pre=0), -1)])
def test_c_entries_refuse_bad_arguments(bad, code):
    L = native.lib()
    a = _args(**bad)
    for entry in (L.vk_block_norm, L.vk_block_norm_backward):
        assert entry(C.byref(a), None) == code
        assert L.vk_last_error().decode().startswith("vk_block_norm")


def test_c_entries_refuse_missing_pointers_overlaps_and_short_workspaces():
    L = native.lib()
    F = lambda **kw: L.vk_block_norm(C.byref(_args(**kw)), None)
    assert F(x=0) == -1 and F(h=0, n=0) == -1 and F(h_cstride=99) == -1 and F(n_bstride=6399) == -1
    B = lambda **kw: L.vk_block_norm_backward(C.byref(_args(**kw)), None)
    assert B(dx=0) == -1 and B(dy=0) == -1 and B(dh=0, dn=0) == -1 and B(h=0) == -1 and B(gate=0) == -1 and B(scale=0) == -1
    assert F(x_cstride=1 << 25) == -2 and B(dy_cstride=1 << 25) == -2            # an item of 2^30 elements or more
    many = dict(batch=1 << 24, length=1, channels=1)                            # more workgroups than a grid holds
    assert F(**many) == -2 and B(**many, workspace=4096, workspace_bytes=1 << 40) == -2
    assert B(dn=0) == -1 and B(dx_cstride=99) == -1 and B(dgate_cstride=99) == -1
    assert B() == -4
    a = _args()
    need = L.vk_block_norm_backward_workspace_bytes(C.byref(a))
    a.workspace, a.workspace_bytes = 4096, need - 4
    assert need > 0 and L.vk_block_norm_backward(C.byref(a), None) == -4
    assert L.vk_block_norm(None, None) == -1 and L.vk_block_norm_backward(None, None) == -1
    assert L.vk_block_norm(C.byref(_args(batch=0, x=0, h=0, n=0)), None) == 0
    assert L.vk_block_norm(C.byref(_args(length=0, x=0, h=0, n=0)), None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 8, 4)
    with pytest.raises(native.NativeError):
        block_norm(x, x)
