"""Bucketed-bias attention at the edges of its definition.  The 64-bit reference and the derived bounds are those of
test_bucket_attention.py."""
import ctypes as C
import math

import pytest
import torch

from test_bucket_attention import _args, assert_within, both, i64, inputs, ref_of
from vits_amd import native
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
