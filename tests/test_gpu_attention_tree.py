"""Attention of drafted tokens over a cache held in 8 bits against its definition in 64 bits."""
import math
import random

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def run(pa, code, olds, counts, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=1, token_major=False, strided=False, ways=None, width=0, small=False, **kw):
    cache = ref.Cache(code, [max(o + n, 0) for o, n in zip(olds, counts)], kv_heads, dim, page, seed, token_major)
    q = queries(sum(counts), heads, dim, dtype, seed + 1, strided)
    ways = dr.ways_of(dr.parents_of(counts, seed, width)) if ways is None else ways
    rows = dr.rows_of(ways, -(-max(counts) // 64))
    print("drafted", code, olds[:4], counts[:4], heads, kv_heads, dim, page, kw, flush=True)
    out, lse = pa.attention_kv8_tree(q, *cache.operands(pa), rows, cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True, **kw)
    (result, norm, magnitude, spread), least = dr.attention_and_least(q, cache, ways, **{k: v for k, v in kw.items() if k in ("window", "scale")})
    expected = (result, norm, magnitude + 2.0 ** 11 * least if small else magnitude, spread)  # (2^-11 of a magnitude is what the check allows)
    ref.check_attention(out, expected, lse)
    return cache, q, rows, out, lse


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_trees_behind_every_kind_of_length(pa, code, dim, page, dtype):  # noqa: F811
    olds = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 257, 1000, 4090]
    run(pa, code, olds, [7, 1, 3, 2, 0, 5, 8, 7, 1, 2, 6, 4, 3, 8, 7], 8, 2, dim, page, dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (16, 1), (24, 3), (32, 4), (40, 2), (48, 1)])
@pytest.mark.parametrize("tokens", [1, 3, 17])
def test_heads_that_share(pa, heads, kv_heads, tokens):  # noqa: F811
    run(pa, "e4m3", [300, 77, 5], [tokens] * 3, heads, kv_heads, 128, 32, strided=True)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 256, 700])
def test_wide_trees(pa, code, dim, window):  # noqa: F811
    run(pa, code, [513, 40, 1700, 0, 300], [256, 40, 130, 65, 1], 6, 2, dim, 16 if dim == 64 else 64, window=window, strided=True)
    run(pa, code, [513, 40, 1700, 0, 300], [150, 129, 0, 64, 33], 6, 2, dim, 32, window=window, width=2)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("tokens", [1, 4, 12, 13, 31, 32, 33, 64, 100])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_rows_of_every_count(pa, code, tokens, group):  # noqa: F811
    run(pa, code, [700, 90, 0], [tokens, max(1, tokens // 2), tokens], 2 * group, 2, 128, 64)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens", [63, 95, 96, 97, 129, 256])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_many_rows_over_short_caches(pa, code, dim, tokens, group):  # noqa: F811
    run(pa, code, [1300], [tokens], 2 * group, 2, dim, 64, strided=True)
    run(pa, code, [300, 0, 33], [tokens, tokens // 3, 1], 2 * group, 2, dim, 16, dtype=torch.float16, width=3)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [16, 48, 96, 112, 192, 240])
def test_heads_of_other_sizes(pa, code, dim):  # noqa: F811
    run(pa, code, [1, 300, 0, 2077], [5, 1, 9, 12], 8, 2, dim, 16, token_major=True)
    assert not pa.last_kernel().startswith("attention_kv8_generic")
    run(pa, code, [90, 300, 0, 3001], [90, 55, 0, 70], 6, 2, dim, 64, dtype=torch.float16, strided=True, window=256)
    assert not pa.last_kernel().startswith("attention_kv8_generic")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [8, 72, 320, 512])
def test_heads_that_only_the_generic_kernel_takes(pa, code, dim):  # noqa: F811
    run(pa, code, [1, 300, 0, 1077], [3, 1, 7, 20], 8, 2, dim, 16, strided=True)
    assert pa.last_kernel() == "attention_kv8_generic"
    run(pa, code, [90, 200], [90, 35], 4, 4, dim, 32, dtype=torch.float16, window=100)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_every_page_size(pa, page):  # noqa: F811
    run(pa, "i8", [700, 255, 256, 257], [9, 1, 3, 7], 8, 2, 128, page)
    run(pa, "e4m3", [700, 255, 256, 257], [200, 255, 17, 2], 8, 2, 128, page)


@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 64, 200])
def test_long_sequences_are_split_and_joined(pa, tokens):  # noqa: F811
    run(pa, "i8", [20011], [tokens], 8, 2, 128, 64)
    run(pa, "e4m3", [9000, 33, 12345], [tokens, min(tokens, 33), tokens], 4, 4, 64, 16, dtype=torch.float16)
    run(pa, "i8", [9000, 33], [tokens, min(tokens, 33)], 4, 1, 128, 16, window=700)
    run(pa, "i8", [9000, 40], [tokens, min(tokens, 33)], 8, 2, 256, 64)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 112, 128, 256])
@pytest.mark.parametrize("tokens", [5, 6, 7, 8, 9, 12, 16, 20])
def test_several_tokens_over_many_keys(pa, code, dim, tokens):  # noqa: F811
    # 40 to 160 rows over more than 64 KB of keys a compute unit
    kv_heads = 4 if dim == 64 else 2
    run(pa, code, [22030, 5, 1200], [tokens, 2, tokens], 8 * kv_heads, kv_heads, dim, 64)
    run(pa, code, [30, 24100, 0], [tokens, tokens, 0], 7 * kv_heads, kv_heads, dim, 128, window=23000)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kw", [{}, {"window": 1500}])
def test_sequences_of_very_different_lengths(pa, code, dim, kw):  # noqa: F811
    run(pa, code, [5104, 0, 130, 3000, 77, 40], [221, 5, 130, 1, 0, 60], 8, 2, dim, 32, **kw)
    run(pa, code, [20, 12011], [20, 70], 8, 2, dim, 16, dtype=torch.float16, **kw)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [33, 64, 65, 130, 200])
def test_batches_of_more_workgroups_than_compute_units(pa, dim, sequences):  # noqa: F811
    rng = random.Random(sequences + dim)
    counts = [rng.choice([0, 1, 2, 4, 4]) for _ in range(sequences)]
    olds = [rng.choice([0, 0, 1, 17, 33, 90, 255, 256, 400, 700, 1040]) for _ in counts]
    counts[sequences // 2], olds[0], counts[0] = 4, 0, 0  # (and a sequence of no tokens at all)
    run(pa, "e4m3", olds, counts, 16, 8, dim, 16)
    assert pa.last_kernel() == "attention_kv8_few"
    # as many tokens each, without cu_tokens
    cache = ref.Cache("i8", [3 + o // 4 for o in olds], 8, dim, 16, 3)
    ways = dr.ways_of(dr.parents_of([3] * sequences, 4))
    q = queries(3 * sequences, 16, dim, torch.bfloat16, 5, False)
    out, lse = pa.attention_kv8_tree(q, *cache.operands(pa), dr.rows_of(ways, 1), want_lse=True)
    ref.check_attention(out, dr.attention(q, cache, ways), lse)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kw", [(256, {}), (256, {"window": 300}), (176, {})])
def test_large_heads_of_many_rows(pa, code, dtype, dim, kw):  # noqa: F811
    """Sequences of a few keys among them: of 60 x 16 x 256 sums some are of codes that are all small, where the 128 that int8 codes are multiplied with shows.  (By
    attention_and_least, 2^-12 of the sum of p s: f16, int8, an element was off by 3.8e-7, of which 5e-8 were beyond the check's 2^-11 of sum p s |code|; s here is
    some 0.9 / 127, so that bound allows 1.7e-6 more.)"""
    rng = random.Random(dim + len(kw))
    counts = [rng.randint(0, 9) for _ in range(60)]
    run(pa, code, [rng.choice([0, 5, 31, 250, 600]) for _ in counts], counts, 16, 2, dim, 16, dtype, strided=True, small=True, **kw)
    run(pa, code, [5000, 300, 4500, 0, 77], [70, 65, 55, 3, 60], 24, 3, dim, 64, dtype, **kw)


@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("counts", [[3, 1, 4], [40, 5, 64], [200, 3, 70], [256, 100, 1]])
def test_any_bits(pa, dim, counts):  # noqa: F811
    """Rows that are no trees': empty ones, which see the older keys alone, or, of sequences that have none, nothing; later tokens; all."""
    rng = random.Random(sum(counts))
    ways = [[rng.choice([set(), {i}, set(range(n)), set(rng.sample(range(n), rng.randrange(n + 1)))]) for i in range(n)] for n in counts]
    ways[1][0] = set()
    cache, q, rows, out, lse = run(pa, "e4m3", [300, 0, 1000], counts, 8, 2, dim, 16, ways=ways)
    at = counts[0]
    assert bool((out[at] == 0).all()) and bool((lse[at] == -math.inf).all())
    run(pa, "i8", [300, 0, 9000], counts, 8, 2, dim, 64, ways=ways, window=400)


@pytest.mark.parametrize("tokens", [5, 70, 200])
def test_bits_behind_the_last_token_and_wider_rows(pa, tokens):  # noqa: F811
    counts = [tokens, 3]
    cache, q, rows, out, lse = run(pa, "i8", [100, 33], counts, 8, 2, 128, 32, seed=5)
    words = rows.shape[1]
    more = torch.full((sum(counts), 4), -1, dtype=torch.int64, device="cuda")
    more[:, :words] = rows
    for nth, n in enumerate(counts):
        at = sum(counts[:nth])
        for w in range(words):
            keep = min(max(n - 64 * w, 0), 64)
            more[at:at + n, w] |= ~(2 ** keep - 1) if keep < 64 else 0
    again, again_lse = pa.attention_kv8_tree(q, *cache.operands(pa), more, cu_tokens=ref.starts(counts), max_tokens=tokens, want_lse=True)
    assert torch.equal(again, out) and torch.equal(again_lse, lse)


@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("tokens", [6, 40, 100])
def test_fewer_tokens_than_were_drafted(pa, dim, tokens):  # noqa: F811
    """A sequence shorter than its tree: the first tokens have no place, and nobody sees them."""
    counts = [tokens, tokens, tokens]
    run(pa, "e4m3", [-1, 2 - tokens, -tokens], counts, 8, 2, dim, 16)


@pytest.mark.parametrize("tokens", [1, 5, 60])
def test_a_chain_is_causal(pa, tokens):  # noqa: F811
    """The bits of a chain are what attention_kv8 sees, to rounding; bit for bit where the same kernel has the same parts."""
    cache = ref.Cache("i8", [5000, 700], 2, 128, 64, 3)
    q = queries(2 * tokens, 8, 128, torch.bfloat16, 4)
    chain = pa.draft_tree(torch.arange(-1, tokens - 1, dtype=torch.int32, device="cuda").repeat(2), 2)
    for kw in ({}, {"window": 300}):
        expected = ref.attention(q, cache, [tokens] * 2, **kw)
        out, lse = pa.attention_kv8_tree(q, *cache.operands(pa), chain, want_lse=True, **kw)
        ref.check_attention(out, expected, lse)


@pytest.mark.parametrize("tokens", [1, 40, 130])
def test_without_room_to_split_the_result_is_the_same_to_rounding(pa, tokens):  # noqa: F811
    import ctypes
    cache = ref.Cache("i8", [5000, 700], 2, 128, 64, 3)
    q = queries(2 * tokens, 8, 128, torch.bfloat16, 4)
    ways = dr.ways_of(dr.parents_of([tokens] * 2, 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    expected = dr.attention(q, cache, ways)
    size = pa.attention_kv8_tree_workspace_bytes(q, cache.k, cache.table, tokens)
    given = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    for kw in ({}, {"workspace": given} if size else {}, {"max_length": 5000}):
        out, lse = pa.attention_kv8_tree(q, *cache.operands(pa), rows, want_lse=True, **kw)
        ref.check_attention(out, expected, lse)
    out = torch.empty_like(q)
    c = pa._kv8_cache("test", *cache.operands(pa))
    rc = pa.lib().ptoamd_attention_kv8_tree(out.data_ptr(), None, ctypes.addressof(c), rows.data_ptr(), rows.shape[1], q.data_ptr(), pa.BF16, 8, 2 * tokens, None,
                                            tokens, 0, q.stride(0), q.stride(1), out.stride(0), out.stride(1), ctypes.c_float(128 ** -0.5), 0, None, 0,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    ref.check_attention(out, expected)


@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_token_major_caches_and_strided_results(pa, code, tokens):  # noqa: F811
    cache = ref.Cache(code, [300, 4000], 4, 128, 32, 5, token_major=True)
    q = queries(2 * tokens, 8, 128, torch.float16, 6, strided=True)
    ways = dr.ways_of(dr.parents_of([tokens] * 2, 6))
    whole = torch.full((2 * tokens, 10, 160), 7.0, dtype=torch.float16, device="cuda")
    out = pa.attention_kv8_tree(q, *cache.operands(pa), dr.rows_of(ways, -(-tokens // 64)), out=whole[:, 1:9, 16:144])
    ref.check_attention(out, dr.attention(q, cache, ways))
    whole[:, 1:9, 16:144] = 7.0  # (nothing beside the result was written)
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("tokens", [2, 20, 90])
@pytest.mark.parametrize("dim", [64, 128, 72])
def test_what_is_not_a_number_stays_where_it_is_seen(pa, tokens, dim):  # noqa: F811
    """NaN scales and entries that are no pages reach the queries that see such a page, and no other: pages of older keys, and those of a drafted token that
    some see; a NaN query its own row only."""
    page, group = 16, 2
    counts, olds = [tokens] * 4, [400 - 16] * 3 + [400]
    ways = [[{i} for i in range(tokens)] for _ in counts]  # (each sees itself)
    cache = ref.Cache("e4m3", [o + n for o, n in zip(olds, counts)], 2, dim, page, 9)
    q = queries(4 * tokens, 2 * group, dim, torch.bfloat16, 10)
    rows = dr.rows_of(ways, -(-tokens // 64))
    good = pa.attention_kv8_tree(q, *cache.operands(pa), rows)
    ref.check_attention(good, dr.attention(q, cache, ways))
    good = good.view(4, tokens, 2 * group, dim)
    cache.k_scale[cache.table[0, 2].long(), 1] = math.nan
    cache.v_scale[cache.table[1, 384 // page].long(), 0] = math.nan  # drafted tokens 0 .. 15
    cache.table[2, 384 // page] = 1 << 20
    out = pa.attention_kv8_tree(q, *cache.operands(pa), rows).view(4, tokens, 2 * group, dim)
    assert bool(out[0, :, group:].isnan().all()) and torch.equal(out[0, :, :group], good[0, :, :group])
    assert bool(out[1, :16, :group].isnan().all()) and torch.equal(out[1, :, group:], good[1, :, group:]) and torch.equal(out[1, 16:], good[1, 16:])
    assert bool(out[2, :16].isnan().all()) and torch.equal(out[2, 16:], good[2, 16:]) and torch.equal(out[3], good[3])
    q.view(4, tokens, 2 * group, dim)[3, 0, 1, 5] = math.nan
    out = pa.attention_kv8_tree(q, *cache.operands(pa), rows).view(4, tokens, 2 * group, dim)
    assert bool(out[3, 0, 1].isnan().all())
    out[3, 0, 1] = good[3, 0, 1]
    assert torch.equal(out[3], good[3])


@pytest.mark.parametrize("tokens", [4, 100])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_scales_far_apart_and_zero(pa, code, tokens):  # noqa: F811
    """Pages whose values differ by 2^24, a page of zeros (scale 0), large scores, among them pages of drafted tokens."""
    cache = ref.Cache(code, [640], 2, 128, 32, 7)
    for b, factor in enumerate([1.0, 2.0 ** -24, 0.0, 2.0 ** 10, 1.0, 2.0 ** -12, 1.0, 1.0, 3.0, 1.0] + [1.0, 0.0, 2.0 ** 6, 2.0 ** -20, 1.0] * 2):
        cache.v_scale[cache.table[0, b].long()] *= factor
        cache.vd[0][b * 32:(b + 1) * 32] *= factor
    q = queries(tokens, 8, 128, torch.bfloat16, 8)
    ways = dr.ways_of(dr.parents_of([tokens], 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    for by in (1.0, 16.0, 1e-3):
        x = q * by
        out, lse = pa.attention_kv8_tree(x, *cache.operands(pa), rows, want_lse=True)
        # (elements that are small in the keys of a row's largest weights, of pages that are 2^10 of others, hold the roundings of those)
        (result, norm, magnitude, spread), least = dr.attention_and_least(x, cache, ways)
        ref.check_attention(out, (result, norm, magnitude + 2.0 ** 11 * least, spread), lse)  # (2^-11 of a magnitude is what the check allows)


@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("counts", [[2, 0, 1], [30, 5, 0], [200, 3, 70]])
def test_padded_batches(pa, dim, counts):  # noqa: F811
    cache = ref.Cache("e4m3", [3000, 70, 5000], 2, dim, 64, 61)
    used, before, behind = sum(counts), 3, 17
    ways = dr.ways_of(dr.parents_of(counts, 6))
    words = -(-max(counts) // 64)
    rows = torch.full((before + used + behind, words), -1, dtype=torch.int64, device="cuda")
    rows[before:before + used] = dr.rows_of(ways, words)
    q = torch.full((before + used + behind, 8, dim), math.nan, dtype=torch.float16, device="cuda")
    q[before:before + used] = queries(used, 8, dim, torch.float16, 62)
    out = torch.full_like(q, 7.0)
    pa.attention_kv8_tree(q, *cache.operands(pa), rows, cu_tokens=ref.starts(counts) + before, max_tokens=max(counts), out=out)
    ref.check_attention(out[before:before + used], dr.attention(q[before:before + used], cache, ways))
    assert bool((out[:before] == 7.0).all()) and bool((out[before + used:] == 7.0).all())


@pytest.mark.parametrize("tokens", [1, 20, 30, 200])
def test_again_on_another_stream_and_captured(pa, tokens):  # noqa: F811
    counts = [tokens, min(tokens, 200)]
    cache, q, rows, out, lse = run(pa, "e4m3", [7000, 400], counts, 8, 2, 128, 64)
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
    side.synchronize()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    other = torch.empty_like(out)
    pa.attention_kv8_tree(q, *cache.operands(pa), rows, **{**kw, "want_lse": False}, stream=side, out=other)
    side.synchronize()
    assert torch.equal(other, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
    for i in range(3):
        q.mul_(1.25)
        rows.copy_(dr.rows_of(dr.ways_of(dr.parents_of(counts, 70 + i)), rows.shape[1]))
        cache.lengths -= 3
        graph.replay()
        eager = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1]), i


def test_the_generic_kernel(pa, monkeypatch):  # noqa: F811
    monkeypatch.setenv("PTOAMD_FORCE_GENERIC", "1")
    pa.reload_options()
    try:
        run(pa, "i8", [300, 70], [3, 70], 8, 2, 128, 32, window=100)
        assert pa.last_kernel() == "attention_kv8_generic"
    finally:
        monkeypatch.delenv("PTOAMD_FORCE_GENERIC")
        pa.reload_options()


def test_random_shapes(pa):  # noqa: F811
    rng = random.Random(5)
    for i in range(40):
        kv = rng.choice([1, 2, 4])
        counts = [rng.choice([0, 1, 2, rng.randrange(1, 33), rng.randrange(1, 257)]) for _ in range(rng.randrange(1, 5))]
        if not sum(counts):
            counts[0] = 1
        olds = [rng.choice([0, rng.randrange(0, 40), rng.randrange(0, 3000)]) for _ in counts]
        run(pa, rng.choice(["i8", "e4m3"]), olds, counts, kv * rng.choice([1, 2, 3, 5, 8]), kv, rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128]),
            rng.choice([torch.bfloat16, torch.float16]), seed=100 + i, width=rng.choice([0, 1, 4]), window=rng.choice([0, 0, rng.randrange(256, 900)]))
