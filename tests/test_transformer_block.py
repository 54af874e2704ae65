"""The operators of a transformer block in one training step, as they are used together: norm, fused projection, attention
with a bucketed bias, projection, the norm after the block with gate, scale and residual, the norm before the next.

Reference: the same step in 64 bits with autograd.  Tolerance: every tensor that an operator stores is off by at most half
a step of its type, r (fp32 2^-24, bf16 2^-8), relative; in fp32 the operators' own sums add some n 2^-24 with n the longest
contraction.  A value of this step passes a chain of at most 12 stored tensors forward and back, and errors of random sign
grow as the root of their number along the chain while the norms divide by deviations of order one, so a tensor's error in
the 2-norm stays below 12 r (bf16: 4.7e-2) and, in fp32, below 12 * n * 2^-24 with n = 160 (1.2e-4)."""
import math

import pytest
import torch
import torch.nn.functional as F

from vits_amd.attention import RelativeBuckets, bucket_attention
from vits_amd.block_norm import block_norm

pytestmark = pytest.mark.gpu


def make(dtype, B, Cn, H, Hk, T, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0: torch.randn(*s, generator=g) * scale
    D = Cn // H
    p = {
        "x": rnd(B, Cn, T), "gate": rnd(B, Cn, 1, scale=0.3) + 1,
        "w_qkv": rnd((H + 2 * Hk) * D, Cn, 1, scale=Cn ** -0.5), "w_out": rnd(Cn, Cn, 1, scale=Cn ** -0.5),
        "bias": rnd(H, 32, scale=0.5), "scale": rnd(Cn, scale=0.1) + 0.5,
        "w1": rnd(Cn, scale=0.1) + 1, "b1": rnd(Cn, scale=0.1), "w2": rnd(Cn, scale=0.1) + 1, "b2": rnd(Cn, scale=0.1),
        "w3": rnd(Cn, scale=0.1) + 1, "b3": rnd(Cn, scale=0.1),
    }
    stored = {"x", "gate", "w_qkv", "w_out"}                     # tensors of the compute type; the rest stays fp32
    p = {k: (v.to(dtype) if k in stored else v).cuda() for k, v in p.items()}
    return p, rnd(B, Cn, T).to(dtype).cuda(), rnd(B, Cn, T).to(dtype).cuda()


def step(p, dh, dn, buckets, H, Hk, lengths, causal):
    _, n = block_norm(p["x"], pre=(p["w1"], p["b1"]), lengths=lengths)
    qkv = F.conv1d(n, p["w_qkv"])
    D = p["x"].shape[1] // H
    att = bucket_attention(qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:], p["bias"], buckets, heads=H, kv_heads=Hk,
                           key_lengths=lengths, query_lengths=lengths, causal=causal)
    y = F.conv1d(att, p["w_out"])
    h, n2 = block_norm(p["x"], y, post=(p["w2"], p["b2"]), gate=p["gate"], scale=p["scale"], pre=(p["w3"], p["b3"]), lengths=lengths)
    return h, n2, ((h.float() * dh.float()).sum() + (n2.float() * dn.float()).sum())


def step64(p, dh, dn, buckets, H, Hk, lengths, causal):
    x = p["x"]
    B, Cn, T = x.shape
    D = Cn // H
    inside = (torch.arange(T) < lengths.view(-1, 1)).unsqueeze(1)
    norm = lambda v, w, b: (F.layer_norm(v.transpose(1, 2), (Cn,), w, b, 1e-5).transpose(1, 2)) * inside
    n = norm(x, p["w1"], p["b1"])
    qkv = F.conv1d(n, p["w_qkv"])
    q, k, v = (t.reshape(B, -1, D, T) for t in (qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:]))
    k, v = k.repeat_interleave(H // Hk, 1), v.repeat_interleave(H // Hk, 1)
    off = torch.arange(T).view(1, T) - torch.arange(T).view(T, 1)
    where = torch.tensor([[buckets.bucket_of(int(o)) for o in row] for row in off])
    s = q.transpose(2, 3) @ k / math.sqrt(D) + p["bias"][:, where]
    ok = inside.unsqueeze(1) & (off <= 0 if causal else torch.ones_like(off, dtype=torch.bool))
    w = torch.softmax(s.masked_fill(~ok, -math.inf), -1)
    att = (w @ v.transpose(2, 3)).transpose(2, 3).reshape(B, Cn, T) * inside
    z = norm(F.conv1d(att, p["w_out"]), p["w2"], p["b2"])
    h = (x + p["scale"].view(1, -1, 1) * p["gate"] * z) * inside
    n2 = norm(h, p["w3"], p["b3"])
    return h, n2, ((h * dh).sum() + (n2 * dn).sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,Cn,H,Hk,T,causal", [(2, 192, 2, 2, 43, False), (3, 160, 4, 2, 131, True)])
def test_training_step_of_a_block(B, Cn, H, Hk, T, causal, dtype):
    buckets = RelativeBuckets(32, 128, bidirectional=not causal)
    lengths = torch.tensor([T - 17 * i for i in range(B)])
    p, dh, dn = make(dtype, B, Cn, H, Hk, T)
    with torch.enable_grad():
        leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
        h, n2, loss = step(leaves, dh, dn, buckets, H, Hk, lengths.cuda(), causal)
        loss.backward()
        exact = {k: v.cpu().double().requires_grad_() for k, v in p.items()}
        h64, n64, loss64 = step64(exact, dh.cpu().double(), dn.cpu().double(), buckets, H, Hk, lengths, causal)
        loss64.backward()
    tol = 12 * 2.0 ** -8 if dtype == torch.bfloat16 else 12 * 160 * 2.0 ** -24
    far = lambda a, b: float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    assert far(h, h64) <= tol and far(n2, n64) <= tol
    for k in p:
        assert leaves[k].grad is not None and far(leaves[k].grad, exact[k].grad) <= tol, (k, far(leaves[k].grad, exact[k].grad))
