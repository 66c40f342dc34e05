"""Attention over a cache held in 8 bits against its definition in 64 bits."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def queries(tokens, heads, dim, dtype, seed, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if strided:  # beside the keys and values of a fused product
        return torch.randn((tokens, heads + 3, dim), generator=g, device="cuda").to(dtype)[:, 1:1 + heads]
    return torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype)


def run(pa, code, lengths, counts, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=1, token_major=False, strided=False, **kw):
    cache = ref.Cache(code, lengths, kv_heads, dim, page, seed, token_major)
    q = queries(sum(counts), heads, dim, dtype, seed + 1, strided)
    print("attention", code, lengths[:4], counts[:4], heads, kv_heads, dim, page, kw, flush=True)
    out, lse = pa.attention_kv8(q, *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True, **kw)
    expected = ref.attention(q, cache, counts, **{k: v for k, v in kw.items() if k in ("causal", "window", "scale")})
    ref.check_attention(out, expected, lse)
    return cache, q, out, lse


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_token_of_sequences_of_every_kind_of_length(pa, code, dim, page, dtype):  # noqa: F811
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 257, 1000, 0, 4097]
    run(pa, code, lengths, [1] * len(lengths), 8, 2, dim, page, dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (16, 1), (24, 3), (32, 4), (40, 2), (48, 1)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_heads_that_share(pa, heads, kv_heads, tokens):  # noqa: F811
    run(pa, "e4m3", [300, 77, 5], [tokens] * 3, heads, kv_heads, 128, 32, strided=True)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 50), (False, 200)])
def test_chunks_and_prompts(pa, code, dim, causal, window):  # noqa: F811
    lengths, counts = [513, 40, 700, 129, 300, 5], [513, 40, 130, 1, 0, 9]  # (the last has queries before its first key)
    run(pa, code, lengths, counts, 6, 2, dim, 16 if dim == 64 else 64, causal=causal, window=window, strided=True)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [16, 48, 80, 96, 112, 192, 240])
@pytest.mark.parametrize("token_major", [False, True])
def test_heads_of_other_sizes(pa, code, dim, token_major):  # noqa: F811
    run(pa, code, [1, 300, 0, 2077], [1] * 4, 8, 2, dim, 16, token_major=token_major)
    assert not pa.last_kernel().startswith("attention_kv8_generic")
    run(pa, code, [9, 300, 40, 2077], [9, 5, 17, 2], 12, 2, dim, 32, dtype=torch.float16, token_major=token_major, strided=True, window=77)
    run(pa, code, [90, 300, 0, 3001], [90, 55, 0, 70], 6, 2, dim, 64, token_major=token_major)
    assert not pa.last_kernel().startswith("attention_kv8_generic")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [8, 72, 320, 512])
def test_heads_that_only_the_generic_kernel_takes(pa, code, dim):  # noqa: F811
    run(pa, code, [1, 300, 0, 1077], [1] * 4, 8, 2, dim, 16, strided=True)
    assert pa.last_kernel() == "attention_kv8_generic"
    run(pa, code, [90, 200], [90, 35], 4, 4, dim, 32, dtype=torch.float16, window=50)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_every_page_size(pa, page):  # noqa: F811
    run(pa, "i8", [700, 255, 256, 257], [1] * 4, 8, 2, 128, page)
    run(pa, "e4m3", [700, 255, 256, 257], [300, 255, 17, 2], 8, 2, 128, page)


@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 64, 200])
def test_long_sequences_are_split_and_joined(pa, tokens):  # noqa: F811
    run(pa, "i8", [20011], [tokens], 8, 2, 128, 64)
    run(pa, "e4m3", [9000, 33, 12345], [tokens, min(tokens, 33), tokens], 4, 4, 64, 16, dtype=torch.float16)
    run(pa, "i8", [9000, 33], [tokens, min(tokens, 33)], 4, 1, 128, 16, window=700)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 112, 128, 256])
@pytest.mark.parametrize("tokens", [5, 6, 7, 8, 9])
def test_several_tokens_over_many_keys(pa, code, dim, tokens):  # noqa: F811
    # 40 to 72 rows over more than 64 KB of keys a compute unit: one to three, or four, tiles of 16 rows a workgroup
    kv_heads = 4 if dim == 64 else 2
    run(pa, code, [22030, 5, 1200], [tokens, 2, tokens], 8 * kv_heads, kv_heads, dim, 64)
    run(pa, code, [30, 24100, 0], [tokens, tokens, 0], 7 * kv_heads, kv_heads, dim, 128, window=23000)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kw", [{}, {"causal": False}, {"window": 1500}])
def test_chunks_over_sequences_of_very_different_lengths(pa, code, dim, kw):  # noqa: F811
    # keys in equal stretches: tiles of rows cut in many parts, whole ones, some without keys, sequences without rows; queries before the first key
    run(pa, code, [5104, 0, 130, 3000, 77, 40], [321, 5, 130, 1, 0, 60], 8, 2, dim, 32, **kw)
    run(pa, code, [20, 12011], [20, 70], 8, 2, dim, 16, dtype=torch.float16, **kw)


@pytest.mark.parametrize("tokens", [1, 40])
def test_without_room_to_split_the_result_is_the_same_to_rounding(pa, tokens):  # noqa: F811
    cache = ref.Cache("i8", [5000, 700], 2, 128, 64, 3)
    q = queries(2 * tokens, 8, 128, torch.bfloat16, 4)
    expected = ref.attention(q, cache, [tokens] * 2)
    size = pa.attention_kv8_workspace_bytes(q, cache.k, cache.table, tokens)
    given = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    for kw in ({}, {"workspace": given} if size else {}, {"max_length": 5000}):
        out, lse = pa.attention_kv8(q, *cache.operands(pa), want_lse=True, **kw)
        ref.check_attention(out, expected, lse)
    out = torch.empty_like(q)
    c = pa._kv8_cache("test", *cache.operands(pa))
    import ctypes
    rc = pa.lib().ptoamd_attention_kv8(out.data_ptr(), None, ctypes.addressof(c), q.data_ptr(), pa.BF16, 8, 2 * tokens, None, tokens, 0, q.stride(0), q.stride(1),
                                       out.stride(0), out.stride(1), ctypes.c_float(128 ** -0.5), 1, 0, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    ref.check_attention(out, expected)


@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_token_major_caches_and_strided_results(pa, code, tokens):  # noqa: F811
    cache = ref.Cache(code, [300, 4000], 4, 128, 32, 5, token_major=True)
    q = queries(2 * tokens, 8, 128, torch.float16, 6, strided=True)
    whole = torch.full((2 * tokens, 10, 160), 7.0, dtype=torch.float16, device="cuda")
    out = pa.attention_kv8(q, *cache.operands(pa), out=whole[:, 1:9, 16:144])
    ref.check_attention(out, ref.attention(q, cache, [tokens] * 2))
    whole[:, 1:9, 16:144] = 7.0  # (nothing beside the result was written)
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("tokens", [1, 100])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_scales_far_apart_and_zero(pa, code, tokens):  # noqa: F811
    """Pages whose values differ by 2^24, a page of zeros (scale 0), large scores: one key takes nearly all the weight."""
    cache = ref.Cache(code, [640], 2, 128, 64, 7)
    for b, factor in enumerate([1.0, 2.0 ** -24, 0.0, 2.0 ** 10, 1.0, 2.0 ** -12, 1.0, 1.0, 3.0, 1.0]):
        cache.v_scale[cache.table[0, b].long()] *= factor
        cache.vd[0][b * 64:(b + 1) * 64] *= factor
    q = queries(tokens, 8, 128, torch.bfloat16, 8)
    for by in (1.0, 16.0, 1e-3):
        x = q * by
        out, lse = pa.attention_kv8(x, *cache.operands(pa), want_lse=True)
        ref.check_attention(out, ref.attention(x, cache, [tokens]), lse)
    # rows of small and of large elements
    x = q * torch.tensor([1e-20, 1.0, 1e6, 1e-3, 0.0, 1.0, 1e3, 1e-6], device="cuda")[None, :, None].to(q.dtype)
    x[..., 0] *= 2.0 ** 12
    out, lse = pa.attention_kv8(x, *cache.operands(pa), want_lse=True, scale=1e-5)
    ref.check_attention(out, ref.attention(x, cache, [tokens], scale=1e-5), lse)


@pytest.mark.parametrize("tokens", [1, 90])
def test_what_is_not_a_number_stays_where_it_is_seen(pa, tokens):  # noqa: F811
    """A NaN scale or a table entry that is no page reaches the queries that see that page, and no other; a NaN query its own row only."""
    cache = ref.Cache("e4m3", [400, 400, 400, 400], 2, 64, 32, 9)
    q = queries(4 * tokens, 4, 64, torch.bfloat16, 10)
    good = pa.attention_kv8(q, *cache.operands(pa))
    cache.k_scale[cache.table[0, 2].long(), 1] = math.nan
    cache.v_scale[cache.table[1, 11].long(), 0] = math.nan
    cache.table[2, 3] = 1 << 20
    out = pa.attention_kv8(q, *cache.operands(pa)).view(4, tokens, 4, 64)
    good = good.view(4, tokens, 4, 64)
    assert bool(out[0, :, 2:].isnan().all()) and torch.equal(out[0, :, :2], good[0, :, :2])
    places = torch.arange(400 - tokens, 400, device="cuda")
    assert bool(out[1, places >= 352][:, :2].isnan().all()) and torch.equal(out[1, :, 2:], good[1, :, 2:])
    assert not bool(out[1, places < 352].isnan().any())
    assert bool(out[2].isnan().all()) and torch.equal(out[3], good[3])
    cache.table[2, 3] = -1
    assert bool(pa.attention_kv8(q, *cache.operands(pa)).view(4, tokens, 4, 64)[2].isnan().all())
    q.view(4, tokens, 4, 64)[3, 0, 1, 5] = math.nan
    out = pa.attention_kv8(q, *cache.operands(pa)).view(4, tokens, 4, 64)
    assert bool(out[3, 0, 1].isnan().all())
    out[3, 0, 1] = good[3, 0, 1]
    assert torch.equal(out[3], good[3])


def test_a_cache_beyond_32_bits(pa):  # noqa: F811
    pages, heads, page, dim = 36000, 8, 128, 128
    k, v = (torch.zeros((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2))
    scale = torch.ones((pages, heads), device="cuda")
    small = ref.Cache("i8", [500, 300], heads, dim, page, 11)
    far = torch.full_like(small.table, -1)
    for s, n in enumerate([500, 300]):
        for b in range(-(-n // page)):
            to, src = pages - 1 - 7 * (4 * s + b), int(small.table[s, b])
            far[s, b] = to
            k[to], v[to] = small.k[src].view(torch.int8), small.v[src].view(torch.int8)
    ks, vs = scale.clone(), scale.clone()
    for s in range(2):
        for b in range(-(-[500, 300][s] // page)):
            ks[far[s, b].long()], vs[far[s, b].long()] = small.k_scale[small.table[s, b].long()], small.v_scale[small.table[s, b].long()]
    for tokens in (1, 100):
        q = queries(2 * tokens, 16, dim, torch.bfloat16, 12)
        out = pa.attention_kv8(q, k, v, ks, vs, far, small.lengths, pa.I8)
        ref.check_attention(out, ref.attention(q, small, [tokens] * 2))
        assert torch.equal(out, pa.attention_kv8(q, *small.operands(pa)))


@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_again_on_another_stream_and_captured(pa, tokens):  # noqa: F811
    cache, q, out, lse = run(pa, "e4m3", [7000, 400], [tokens, min(tokens, 300)], 8, 2, 128, 64)
    counts = [tokens, min(tokens, 300)]
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = pa.attention_kv8(q, *cache.operands(pa), **kw)
    side.synchronize()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pa.attention_kv8(q, *cache.operands(pa), **kw)
    for i in range(3):
        q.mul_(1.25)
        graph.replay()
        eager = pa.attention_kv8(q, *cache.operands(pa), **kw)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1]), i


def test_the_generic_kernel(pa, monkeypatch):  # noqa: F811
    monkeypatch.setenv("PTOAMD_FORCE_GENERIC", "1")
    pa.reload_options()
    try:
        run(pa, "i8", [300, 70], [3, 70], 8, 2, 128, 32)
        assert pa.last_kernel() == "attention_kv8_generic"
    finally:
        monkeypatch.delenv("PTOAMD_FORCE_GENERIC")
        pa.reload_options()
    run(pa, "e4m3", [300, 70], [3, 70], 8, 2, 8, 32)
    run(pa, "e4m3", [300, 70], [3, 70], 4, 2, 512, 32)
    assert pa.last_kernel() == "attention_kv8_generic"


def test_random_shapes(pa):  # noqa: F811
    import random
    rng = random.Random(5)
    for i in range(30):
        kv = rng.choice([1, 2, 4])
        counts = [rng.choice([0, 1, 1, 2, rng.randrange(1, 150)]) for _ in range(rng.randrange(1, 5))]
        if not sum(counts):
            counts[0] = 1
        lengths = [max(1, n + rng.choice([0, -1, rng.randrange(0, 40), rng.randrange(0, 3000)])) for n in counts]
        run(pa, rng.choice(["i8", "e4m3"]), lengths, counts, kv * rng.choice([1, 2, 3, 5, 8]), kv, rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128]),
            rng.choice([torch.bfloat16, torch.float16]), seed=100 + i, causal=rng.random() < 0.8, window=rng.choice([0, 0, rng.randrange(1, 300)]))
