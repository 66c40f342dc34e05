"""Batches padded to a captured size: rows that no sequence has are neither read nor written."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("counts", [[1, 0, 1], [30, 5, 0], [200, 3, 70]])
def test_attention_leaves_them_alone(pa, dim, counts):  # noqa: F811
    cache = ref.Cache("e4m3", [3000, 70, 5000], 2, dim, 64, 61)
    used, before, behind = sum(counts), 3, 17
    q = torch.full((before + used + behind, 8, dim), math.nan, dtype=torch.float16, device="cuda")
    q[before:before + used] = queries(used, 8, dim, torch.float16, 62)
    out = torch.full_like(q, 7.0)
    pa.attention_kv8(q, *cache.operands(pa), cu_tokens=ref.starts(counts) + before, max_tokens=max(counts), out=out)
    ref.check_attention(out[before:before + used], ref.attention(q[before:before + used], cache, counts))
    assert bool((out[:before] == 7.0).all()) and bool((out[before + used:] == 7.0).all())
    # beyond max_tokens: the first ones of each sequence alone, at their places
    out.fill_(7.0)
    most = max(counts) - 1
    pa.attention_kv8(q, *cache.operands(pa), cu_tokens=ref.starts(counts) + before, max_tokens=most, out=out)
    at = before
    for n in counts:
        assert bool((out[at + min(n, most):at + n] == 7.0).all())
        at += n


def test_the_append_does_not_read_them(pa):  # noqa: F811
    counts = [3, 0, 40]
    caches = [ref.Cache("i8", [30, 20, 90], 2, 64, 16, 63) for _ in range(2)]
    k, v = queries(43, 2, 64, torch.bfloat16, 64), queries(43, 2, 64, torch.bfloat16, 65)
    wide = [torch.full((60, 2, 64), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for to, x in zip(wide, (k, v)):
        to[5:48] = x
    pa.kvcache_append(k, v, *caches[0].operands(pa), cu_tokens=ref.starts(counts), max_tokens=40)
    pa.kvcache_append(*wide, *caches[1].operands(pa), cu_tokens=ref.starts(counts) + 5, max_tokens=40)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8)), name
