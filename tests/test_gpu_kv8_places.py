"""Attention over an 8-bit cache where queries stand before the first key and windows are as long as 32 bits hold."""
import pytest
import torch

import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tokens", [3, 20, 300])
@pytest.mark.parametrize("dim", [64, 128, 256, 72])
def test_a_window_beyond_every_key_hides_none(pa, dim, tokens, causal, window):  # noqa: F811
    """As without a window, bit for bit, idle sequences (no key, but queries) and queries before the first key among them."""
    cache = ref.Cache("e4m3", [0, 2, 700, 5000], 2, dim, 64, 31)
    counts = [tokens, tokens, tokens, 1]
    q = queries(sum(counts), 8, dim, torch.bfloat16, 32)
    print("window", dim, tokens, causal, window, flush=True)
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=tokens, causal=causal, want_lse=True)
    plain = pa.attention_kv8(q, *cache.operands(pa), **kw)
    ref.check_attention(plain[0], ref.attention(q, cache, counts, causal=causal), plain[1])
    got = pa.attention_kv8(q, *cache.operands(pa), window=window, **kw)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


@pytest.mark.parametrize("most", [101, 2 ** 20, 2 ** 31 - 1])
def test_a_loose_bound_of_the_new_tokens(pa, most):  # noqa: F811
    """max_tokens may be more than any sequence has, and more than all have together."""
    counts = [5, 1, 95]
    for heads in (2, 16):
        caches = [ref.Cache("i8", [40, 700, 300], 2, 128, 64, 33) for _ in range(2)]
        q = queries(sum(counts), heads, 128, torch.bfloat16, 34)
        k, v = queries(sum(counts), 2, 128, torch.bfloat16, 35), queries(sum(counts), 2, 128, torch.bfloat16, 36)
        outs = []
        for cache, bound in zip(caches, (95, most)):
            print("bound", heads, bound, flush=True)
            pa.kvcache_append(k, v, *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=bound)
            outs.append(pa.attention_kv8(q, *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=bound, want_lse=True))
            outs[-1] += (pa.attention_kv8(q[:3], *cache.operands(pa), cu_tokens=ref.starts([1, 1, 1]), max_tokens=1 if bound == 95 else bound),)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8)), name
        for a, b in zip(*outs):  # (another bound may take another kernel: the same but for rounding, an f16 weight's and a bf16 result's)
            assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * a.double().abs().max()).all())
