"""A block table entry that is no page reaches the queries that see it and no other, whatever the cache holds beside it."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 112, 128, 256, 72])
@pytest.mark.parametrize("tokens,heads", [(5, 2), (20, 2), (100, 8)])
@pytest.mark.parametrize("entry", [-1, 1 << 20])
@pytest.mark.parametrize("scale", [1.0, math.inf, math.nan, 0.0])
def test_an_entry_that_only_later_queries_see(pa, dim, tokens, heads, entry, scale):  # noqa: F811
    """The last page of a sequence, whose first place is in the middle of the new tokens, is none; page 0, which nothing names, holds NaN codes under
    any scale."""
    page = 16
    length = 320 + tokens // 2
    cache = ref.Cache("e4m3", [length, 300], 2, dim, page, 41)
    for name in ("k", "v"):  # (a page of NaN codes in front of the others)
        codes, scales = getattr(cache, name), getattr(cache, name + "_scale")
        setattr(cache, name, torch.cat([torch.full_like(codes[:1], 0x7F), codes]))
        setattr(cache, name + "_scale", torch.cat([torch.full_like(scales[:1], scale), scales]))
    cache.table = torch.where(cache.table < 0, cache.table, cache.table + 1)
    q = queries(2 * tokens, heads, dim, torch.bfloat16, 42)
    expected = ref.attention(q, cache, [tokens] * 2)
    at = 320 // page
    cache.table[0, at] = entry
    print("unknown page", dim, tokens, heads, entry, scale, flush=True)
    out, lse = pa.attention_kv8(q, *cache.operands(pa), want_lse=True)
    sees = torch.arange(length - tokens, length, device="cuda") >= 320
    assert 0 < int(sees.sum()) < tokens
    mine = torch.cat([sees, torch.zeros_like(sees)])
    assert bool(out[mine].isnan().all()) and bool(lse[mine].isnan().all())
    ref.check_attention(out[~mine], [x[~mine] for x in expected], lse[~mine])
