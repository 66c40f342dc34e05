"""Chains of drafted tokens against attention_kv8, keys of the append with rotation against the rotation in 64 bits, int8 values of few small codes."""
import math

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_append_rope import fused, places
from test_gpu_attention_kv8 import queries
from test_gpu_kvcache_append import grown, snapshot
from test_gpu_parity import pa  # noqa: F401
from test_gpu_rope import turned

pytestmark = pytest.mark.gpu


# ---- chains ---------------------------------------------------------------------------------------------------------------
def both(pa, cache, q, counts, **kw):  # noqa: F811
    """A chain's bits on attention_kv8_tree, and attention_kv8 of the same tokens, each with the kernel that ran."""
    parents = torch.tensor([i - 1 for n in counts for i in range(n)], dtype=torch.int32, device="cuda")
    chain = pa.draft_tree(parents, len(counts), cu_tokens=ref.starts(counts), max_tokens=max(counts))
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True, **kw)
    got = pa.attention_kv8_tree(q, *cache.operands(pa), chain, **kw)
    kernel = pa.last_kernel()
    want = pa.attention_kv8(q, *cache.operands(pa), causal=True, **kw)
    assert pa.last_kernel() == kernel, (pa.last_kernel(), kernel)
    return got, want, kernel


@pytest.mark.parametrize("window", [0, 256])
@pytest.mark.parametrize("kernel,dim,kv_heads,group,tokens,olds", [
    ("attention_kv8_few", 64, 2, 4, 3, [600, 0, 33, 255]), ("attention_kv8_few", 128, 2, 16, 1, [600, 0, 33, 255]), ("attention_kv8_few", 112, 4, 2, 7, [640, 5, 31, 64]),
    ("attention_kv8_many", 64, 8, 3, 70, [300, 0, 31, 64, 129, 200, 90] * 3), ("attention_kv8_many", 128, 8, 3, 70, [300, 0, 31, 64, 129, 200, 90] * 3),
    ("attention_kv8_many", 256, 8, 3, 70, [300, 0, 31, 64, 129, 200, 90] * 7)])
def test_a_chain_is_causal_bit_for_bit(pa, kernel, dim, kv_heads, group, tokens, olds, window):  # noqa: F811
    """E4M3, the same kernel with the same keys a workgroup: the same products and sums, and keys that a row does not see add zeros.  (With a window, a second tile of rows,
    which heads of 256 have here from 128 rows on, starts at its first row's first key in attention_kv8, where a tree has the sequence's: other tiles of keys, so
    other references; both are within their bounds.)"""
    counts = [tokens] * len(olds)
    counts[1] = 1
    cache = ref.Cache("e4m3", [o + n for o, n in zip(olds, counts)], kv_heads, dim, 64, 5)
    q = queries(sum(counts), kv_heads * group, dim, torch.bfloat16, 6)
    got, want, ran = both(pa, cache, q, counts, window=window)
    assert ran == kernel
    for out, lse in (got, want):
        ref.check_attention(out, ref.attention(q, cache, counts, window=window), lse)
    same_keys = window == 0 or kernel != "attention_kv8_many" or tokens * group <= (128 if dim == 256 else 256)
    assert not same_keys or (torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]))


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("window", [0, 100])
def test_a_chain_is_causal_on_the_generic_kernel(pa, monkeypatch, code, window):  # noqa: F811
    monkeypatch.setenv("PTOAMD_FORCE_GENERIC", "1")
    pa.reload_options()
    try:
        counts = [90, 1, 33]
        cache = ref.Cache(code, [300 + 90, 1, 70 + 33], 2, 72, 32, 5)
        q = queries(sum(counts), 6, 72, torch.float16, 6)
        got, want, ran = both(pa, cache, q, counts, window=window)
        assert ran == "attention_kv8_generic"
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    finally:
        monkeypatch.delenv("PTOAMD_FORCE_GENERIC")
        pa.reload_options()


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 5, 60, 200])
def test_a_chain_is_causal_to_rounding(pa, code, dim, tokens):  # noqa: F811
    """Whatever kernels and parts the two take: each within its bound of the result in 64 bits."""
    cache = ref.Cache(code, [5000, 700], 2, dim, 64, 3)
    q = queries(2 * tokens, 8, dim, torch.bfloat16, 4)
    ways = [[set(range(i + 1)) for i in range(tokens)] for _ in range(2)]
    rows = dr.rows_of(ways, -(-tokens // 64))
    for kw in ({}, {"window": 300}):
        (out, norm, magnitude, spread), least = dr.attention_and_least(q, cache, ways, **kw)
        for call, args in ((pa.attention_kv8_tree, (rows,)), (pa.attention_kv8, ())):
            got, lse = call(q, *cache.operands(pa), *args, want_lse=True, **kw)
            ref.check_attention(got, (out, norm, magnitude + 2.0 ** 11 * least, spread), lse)


@pytest.mark.parametrize("tokens", [1, 5, 40, 150])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_int8_values_of_few_small_codes(pa, dim, tokens):  # noqa: F811
    """Values whose codes are 0 but for a few of 1 or -1: what the 128 that codes are multiplied with leaves behind is within 2^-12 of the sum of weight times scale
    (attention_and_least), of both calls."""
    cache = ref.Cache("i8", [900, 64 + tokens], 2, dim, 64, 3)
    g = torch.Generator(device="cuda").manual_seed(9)
    for s, n in enumerate(cache.lengths.tolist()):
        for b in range(-(-n // 64)):
            page, held = int(cache.table[s, b]), min(n, 64 * (b + 1)) - 64 * b
            codes = (torch.randint(0, 50, (2, held, dim), generator=g, device="cuda") == 0) * (2 * torch.randint(0, 2, (2, held, dim), generator=g, device="cuda") - 1)
            cache.v[page, :, :held] = codes.to(torch.int8).view(torch.uint8)
            cache.vd[s][64 * b:64 * b + held] = codes.double().transpose(0, 1) * cache.v_scale[page].double()[:, None]
    q = queries(2 * tokens, 8, dim, torch.float16, 4)
    ways = [[set(range(i + 1)) for i in range(tokens)] for _ in range(2)]
    rows = dr.rows_of(ways, -(-tokens // 64))
    (out, norm, magnitude, spread), least = dr.attention_and_least(q, cache, ways)
    for call, args in ((pa.attention_kv8_tree, (rows,)), (pa.attention_kv8, ())):
        got, lse = call(q, *cache.operands(pa), *args, want_lse=True)
        print("beside 2^-11 of the magnitude:", float(((got.double() - out).abs() - 2.0 ** -11 * (out.abs() + magnitude)).max() / least.max()), flush=True)
        ref.check_attention(got, (out, norm, magnitude + 2.0 ** 11 * least, spread), lse)


# ---- keys -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (96, 24), (80, 20)])
@pytest.mark.parametrize("tree", [False, True])
def test_keys_turned_in_64_bits(pa, code, dtype, interleaved, dim, rot, tree):  # noqa: F811
    """Two products and their sum, each rounded to f32: a rotated element is off by `off` = 2^-23 of |a cos| + |b sin|.  A scale is the largest of them times 1 / Q, two
    roundings: within off / Q and 2^-23 of itself.  A code is the nearest to x * (1 / scale), two roundings: half a step, off / scale and 2^-23 of itself, twice that
    allowed; a step's size goes by the value in 64 bits, and one that the roundings lift over a power of two lies as near to that."""
    olds, counts, page, heads = [0, 17, 40, 64], [50, 3, 90, 1], 32, 2
    parents = dr.parents_of(counts, 7)
    ways = dr.ways_of(parents)
    positions = places(olds, counts)
    if tree:
        positions = torch.tensor([o + len(w) - 1 for o, mine in zip(olds, ways) for w in mine], dtype=torch.int32, device="cuda")
    table = pa.rope_table(300, rot)
    q, k, v = fused(sum(counts), 4, heads, dim, dtype, 3)
    cache = grown(code, olds, counts, heads, dim, page, 6)
    before = snapshot(cache)
    got = pa.kvcache_append_rope(q, k, v, *cache.operands(pa), table, tree=dr.rows_of(ways, 2) if tree else None, interleaved=interleaved, cu_tokens=ref.starts(counts),
                                 max_tokens=90)
    exact, size = turned(q, table, positions, interleaved, False)
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    assert bool(((got.double() - exact).abs() <= unit * exact.abs() * (1 + 2.0 ** -10) + 2.0 ** -23 * size + (2.0 ** -24 if dtype == torch.float16 else 0.0)).all())
    keys, size = turned(k, table, positions, interleaved, False)
    largest = ref.LARGEST[code]
    for name, x, off in (("k", keys, 2.0 ** -23 * size), ("v", v.double(), torch.zeros_like(v, dtype=torch.float64))):
        codes, scales, at = getattr(cache, name), getattr(cache, name + "_scale"), 0
        for s, (old, n) in enumerate(zip(olds, counts)):
            for b in range(old // page, -(-(old + n) // page)):
                lo, hi, its = max(old, b * page), min(old + n, (b + 1) * page), int(cache.table[s, b])
                older = lo - b * page
                rows, far = (t[at + lo - old:at + hi - old].transpose(0, 1) for t in (x, off))
                now, most = scales[its].double(), rows.abs().amax(dim=(1, 2)) / largest
                held = before[name + "_scale"][its].double() if older else torch.zeros_like(now)
                slack = far.amax(dim=(1, 2)) / largest + 2.0 ** -23 * most
                assert bool((now >= torch.maximum(held, most - slack)).all()) and bool((now <= torch.maximum(held, most + slack)).all()), (name, s, b)
                want = rows / now[:, None, None]
                step = 1.0 if code == "i8" else torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -6))) - 3)
                tol = 0.5 * step + 2 * (far / now[:, None, None] + 2.0 ** -23 * want.abs())
                mine = ref.code_values(codes[its, :, older:older + hi - lo].contiguous(), code)
                assert bool(((mine - want).abs() <= tol).all()), (name, s, b, float(((mine - want).abs() - tol).max()))
            at += n
