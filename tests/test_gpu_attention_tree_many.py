"""Attention of drafted tokens on the many-rows kernel: up to 128 rows of a key head as two halves that share their rows, more as tiles of 256 (128 of heads of 256);
keys whole and in stretches that are joined.  Every call asserts that this kernel ran.  (How far results may be off: drafted_reference.attention_and_least.)"""
import ctypes
import math
import random
import types

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu

WHOLE, CUT = "attention_kv8_many", "attention_kv8_many_split"
WIDE = 120000  # tokens of a table that plans for keys in stretches
OLDS = [0, 1, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 191, 193, 200, 255, 257, 300, 320, 383, 400, 410, 0, 17, 90, 254, 256, 350, 5, 77, 150, 222, 303]
# (tokens drafted for a sequence at the most, query heads a key head): 66, 128, 128 rows, two halves; 160, 300, 512
FORMS = [(11, 6), (32, 4), (16, 8), (40, 4), (100, 3), (256, 2)]


def widened(cache, tokens):
    """The cache with a table of that many tokens' pages, of which the sequences have what they had."""
    blocks = tokens // cache.page - cache.table.shape[1]
    if blocks > 0:
        cache.table = torch.cat([cache.table, torch.full((cache.table.shape[0], blocks), -7, dtype=torch.int32, device="cuda")], dim=1)
    return cache


def expected_of(q, cache, ways, **kw):
    (out, norm, magnitude, spread), least = dr.attention_and_least(q, cache, ways, **kw)
    return out, norm, magnitude + 2.0 ** 11 * least, spread  # (2^-11 of a magnitude is what the check allows)


def call(pa, kernel, q, cache, rows, counts, **kw):  # noqa: F811
    got = pa.attention_kv8_tree(q, *cache.operands(pa), rows, cu_tokens=ref.starts(counts), max_tokens=max(counts), **{"want_lse": True, **kw})
    assert pa.last_kernel() == kernel, pa.last_kernel()
    return got


def run(pa, kernel, code, olds, counts, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=1, token_major=False, strided=False, ways=None, width=0, wide=0, **kw):  # noqa: F811
    cache = widened(ref.Cache(code, [max(o + n, 0) for o, n in zip(olds, counts)], kv_heads, dim, page, seed, token_major), wide)
    q = queries(sum(counts), heads, dim, dtype, seed + 1, strided)
    ways = dr.ways_of(dr.parents_of(counts, seed, width)) if ways is None else ways
    rows = dr.rows_of(ways, -(-max(counts) // 64))
    print("drafted, many rows", kernel, code, olds[:4], counts[:4], heads, kv_heads, dim, page, wide, kw, flush=True)
    out, lse = call(pa, kernel, q, cache, rows, counts, **kw)
    ref.check_attention(out, expected_of(q, cache, ways, **{k: v for k, v in kw.items() if k in ("window", "scale")}), lse)
    return cache, q, ways, rows, out, lse


def batch(tokens, seed, sequences=33):
    """Ragged counts of a batch, none and one token among them."""
    rng = random.Random(seed)
    counts = [rng.randint(max(1, 3 * tokens // 4), tokens) for _ in range(sequences)]
    counts[1], counts[4], counts[7] = tokens, 0, 1
    return counts


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 80, 112, 128])
@pytest.mark.parametrize("tokens,group", FORMS)
def test_batches(pa, code, dim, tokens, group, wide):  # noqa: F811
    """Of many sequences: a workgroup a tile of rows, or, of a wide table, stretches that hold the ends and starts of several."""
    few = tokens > 64
    counts = batch(tokens, tokens + dim, 12 if few else 33)
    run(pa, CUT if wide else WHOLE, code, OLDS[:len(counts)], counts, 8 * group, 8, dim, 16 if dim == 64 else 32, strided=True, wide=wide,
        dtype=torch.float16 if dim == 112 else torch.bfloat16, width=3 if few else 0)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,group", FORMS + [(65, 1), (128, 1), (129, 1)])
def test_a_few_sequences_in_many_stretches(pa, code, dim, tokens, group):  # noqa: F811
    """Tiles of rows in many parts, a short sequence whole beside them, one without rows; the second half's tiles one fewer or as many."""
    for olds in ([5003, 64, 300], [4097, 0, 640], [3967, 129, 2000]):
        run(pa, CUT, code, olds, [tokens, max(1, tokens // 3), 0], 2 * group, 2, dim, 64, dtype=torch.float16, wide=2 ** 20, seed=olds[0])


@pytest.mark.parametrize("tokens,group", FORMS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,kernel", [(256, WHOLE), (12000, CUT)])
def test_windows(pa, dim, tokens, group, window, kernel):  # noqa: F811
    olds = [700, 0, 255, 256, 257, 3100, 4000, 90, 300, 330, 12990, 12003, 1024, 600, 5, 64, 3500]
    counts = batch(tokens, tokens, len(olds))
    kv_heads = 8 if kernel == CUT else 32 if (tokens, group) == (11, 6) else 16  # (whole: more workgroups than the few-rows kernel takes)
    run(pa, kernel, "e4m3", olds, counts, kv_heads * group, kv_heads, dim, 64, window=window, wide=WIDE)


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,group", FORMS)
def test_any_bits(pa, dim, tokens, group, wide):  # noqa: F811
    """Rows that are no trees', empty ones among them, sequences without older keys, rows wider than they need be with bits behind the last token."""
    rng = random.Random(tokens)
    counts = batch(tokens, tokens + 1, 12 if tokens > 64 else 33)
    ways = [[rng.choice([set(), {i}, set(range(n)), set(rng.sample(range(n), rng.randrange(n + 1)))]) for i in range(n)] for n in counts]
    olds = OLDS[:len(counts)]
    olds[1], ways[1][0] = 0, set()
    cache, q, ways, rows, out, lse = run(pa, CUT if wide else WHOLE, "i8", olds, counts, 8 * group, 8, dim, 16, ways=ways, wide=wide)
    at = counts[0]
    assert bool((out[at] == 0).all()) and bool((lse[at] == -math.inf).all())
    more = torch.full((sum(counts), 4), -1, dtype=torch.int64, device="cuda")
    words, at = rows.shape[1], 0
    more[:, :words] = rows
    for n in counts:
        for w in range(words):
            keep = min(max(n - 64 * w, 0), 64)
            more[at:at + n, w] |= ~(2 ** keep - 1) if keep < 64 else 0
        at += n
    again, again_lse = call(pa, CUT if wide else WHOLE, q, cache, more, counts)
    assert torch.equal(again, out) and torch.equal(again_lse, lse)


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("dim", [64, 112, 128])
@pytest.mark.parametrize("tokens,group", [(32, 4), (40, 4)])
def test_what_is_not_a_number_stays_where_it_is_seen(pa, tokens, dim, group, wide):  # noqa: F811
    """NaN scales and entries that are no pages reach the queries that see such a page, and no other."""
    page, kv, seqs = 16, 8, 33
    counts, old = [tokens] * seqs, 368
    ways = [[{i} for i in range(tokens)] for _ in counts]  # (each sees itself)
    cache = widened(ref.Cache("e4m3", [old + tokens] * seqs, kv, dim, page, 9), wide)
    q = queries(seqs * tokens, kv * group, dim, torch.bfloat16, 10)
    rows = dr.rows_of(ways, 1)
    kernel = CUT if wide else WHOLE
    shape = (seqs, tokens, kv * group, dim)
    good, expected = call(pa, kernel, q, cache, rows, counts, want_lse=False), expected_of(q, cache, ways)
    ref.check_attention(good, expected)
    good = good.view(shape)
    cache.k_scale[cache.table[0, 2].long(), 1] = math.nan
    cache.v_scale[cache.table[1, 384 // page].long(), 0] = math.nan  # drafted tokens 16 .. 31
    cache.table[2, 384 // page] = 1 << 20
    cache.table[seqs - 1, 5] = -1
    out = call(pa, kernel, q, cache, rows, counts, want_lse=False).view(shape)
    its = slice(group, 2 * group)
    assert bool(out[0, :, its].isnan().all()) and torch.equal(out[0, :, :group], good[0, :, :group]) and torch.equal(out[0, :, 2 * group:], good[0, :, 2 * group:])
    assert bool(out[1, 16:32, :group].isnan().all()) and torch.equal(out[1, :, group:], good[1, :, group:])
    assert torch.equal(out[1, :16], good[1, :16]) and torch.equal(out[1, 32:], good[1, 32:])
    assert bool(out[2, 16:32].isnan().all()) and torch.equal(out[2, :16], good[2, :16]) and torch.equal(out[2, 32:], good[2, 32:])
    assert torch.equal(out[3:-1], good[3:-1]) and bool(out[-1].isnan().all())
    q.view(shape)[3, 5, 1, 7] = math.nan
    q.view(shape)[4, 6, 2, 3] = math.inf
    out = call(pa, kernel, q, cache, rows, counts, want_lse=False).view(shape)
    assert bool(out[3, 5, 1].isnan().all()) and bool(out[4, 6, 2].isnan().all())
    out[3, 5, 1], out[4, 6, 2] = good[3, 5, 1], good[4, 6, 2]
    assert torch.equal(out[5:-1], good[5:-1])
    # (rows of the same wave: their references may follow others' largest scores, so not bit for bit)
    ref.check_attention(out[3:5].flatten(0, 1), [x[3 * tokens:5 * tokens] for x in expected])


@pytest.mark.parametrize("tokens,group", FORMS)
@pytest.mark.parametrize("dim", [64, 128])
def test_stretches_without_a_workspace_and_with_a_given_one(pa, dim, tokens, group):  # noqa: F811
    cache = widened(ref.Cache("i8", [3000 + tokens, 70 + tokens], 2, dim, 64, 3), 2 ** 20)
    q = queries(2 * tokens, 2 * group, dim, torch.bfloat16, 4)
    ways = dr.ways_of(dr.parents_of([tokens] * 2, 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    expected = expected_of(q, cache, ways)
    given = torch.empty(pa.attention_kv8_tree_workspace_bytes(q, cache.k, cache.table, tokens), dtype=torch.uint8, device="cuda")
    ref.check_attention(call(pa, CUT, q, cache, rows, [tokens] * 2, workspace=given, want_lse=False), expected)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    c = pa._kv8_cache("test", *cache.operands(pa))
    rc = pa.lib().ptoamd_attention_kv8_tree(out.data_ptr(), lse.data_ptr(), ctypes.addressof(c), rows.data_ptr(), rows.shape[1], q.data_ptr(), pa.BF16, 2 * group,
                                            2 * tokens, None, tokens, 0, q.stride(0), q.stride(1), out.stride(0), out.stride(1), ctypes.c_float(dim ** -0.5), 0, None, 0,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and pa.last_kernel() == WHOLE
    ref.check_attention(out, expected, lse)


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("tokens,group", [(32, 4), (100, 3)])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_token_major_caches_and_strided_results(pa, code, tokens, group, wide):  # noqa: F811
    counts = batch(tokens, 3, 12 if tokens > 64 else 33)
    cache = widened(ref.Cache(code, [o + n for o, n in zip(OLDS, counts)], 8, 128, 32, 5, token_major=True), wide)
    q = queries(sum(counts), 8 * group, 128, torch.float16, 6, strided=True)
    ways = dr.ways_of(dr.parents_of(counts, 6))
    expected = expected_of(q, cache, ways)
    for off in (16, 3):  # (on 16 bytes, and not)
        whole = torch.full((sum(counts), 8 * group + 2, 160), 7.0, dtype=torch.float16, device="cuda")
        out = whole[:, 1:-1, off:off + 128]
        call(pa, CUT if wide else WHOLE, q, cache, dr.rows_of(ways, -(-tokens // 64)), counts, out=out, want_lse=False)
        ref.check_attention(out, expected)
        out.fill_(7.0)  # (nothing beside the result was written)
        assert bool((whole == 7.0).all())


@pytest.mark.parametrize("tokens,group", [(20, 4), (80, 4)])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_scales_far_apart_and_zero(pa, code, tokens, group):  # noqa: F811
    """Pages whose values differ by 2^24, a page of zeros (scale 0), large scores, among them pages of drafted tokens."""
    cache = widened(ref.Cache(code, [640], 2, 128, 32, 7), 2 ** 20)
    for b, factor in enumerate([1.0, 2.0 ** -24, 0.0, 2.0 ** 10, 1.0, 2.0 ** -12, 1.0, 1.0, 3.0, 1.0] + [1.0, 0.0, 2.0 ** 6, 2.0 ** -20, 1.0] * 2):
        cache.v_scale[cache.table[0, b].long()] *= factor
        cache.vd[0][b * 32:(b + 1) * 32] *= factor
    q = queries(tokens, 2 * group, 128, torch.bfloat16, 8)
    ways = dr.ways_of(dr.parents_of([tokens], 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    for by in (1.0, 16.0, 1e-3):
        out, lse = call(pa, CUT, q * by, cache, rows, [tokens])
        ref.check_attention(out, expected_of(q * by, cache, ways), lse)


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,group", [(32, 4), (40, 4), (100, 3)])
def test_fewer_tokens_than_were_drafted(pa, dim, tokens, group, wide):  # noqa: F811
    """Sequences shorter than their trees: the first tokens have no place, and nobody sees them."""
    seqs = 33 if tokens < 64 else 12
    olds = [(-1, 2 - tokens, -tokens, -tokens // 2, 100)[i % 5] for i in range(seqs)]
    run(pa, CUT if wide else WHOLE, "e4m3", olds, [tokens] * seqs, 8 * group, 8, dim, 16, wide=wide)


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,group", [(32, 4), (100, 3)])
def test_padded_batches(pa, dim, tokens, group, wide):  # noqa: F811
    counts = batch(tokens, 8, 12 if tokens > 64 else 33)
    cache = widened(ref.Cache("e4m3", [o + n for o, n in zip(OLDS, counts)], 8, dim, 64, 61), wide)
    used, before, behind = sum(counts), 3, 17
    ways = dr.ways_of(dr.parents_of(counts, 6))
    words = -(-tokens // 64)
    rows = torch.full((before + used + behind, words), -1, dtype=torch.int64, device="cuda")
    rows[before:before + used] = dr.rows_of(ways, words)
    q = torch.full((before + used + behind, 8 * group, dim), math.nan, dtype=torch.float16, device="cuda")
    q[before:before + used] = queries(used, 8 * group, dim, torch.float16, 62)
    out = torch.full_like(q, 7.0)
    pa.attention_kv8_tree(q, *cache.operands(pa), rows, cu_tokens=ref.starts(counts) + before, max_tokens=tokens, out=out)
    assert pa.last_kernel() == (CUT if wide else WHOLE)
    ref.check_attention(out[before:before + used], expected_of(q[before:before + used], cache, ways))
    assert bool((out[:before] == 7.0).all()) and bool((out[before + used:] == 7.0).all())


@pytest.mark.parametrize("wide", [0, WIDE])
@pytest.mark.parametrize("tokens,group", [(32, 4), (40, 4), (100, 3)])
def test_again_on_another_stream_and_captured(pa, tokens, group, wide):  # noqa: F811
    kernel = CUT if wide else WHOLE
    counts = batch(tokens, 9, 12 if tokens > 64 else 33)
    cache, q, ways, rows, out, lse = run(pa, kernel, "e4m3", [o + 9 for o in OLDS[:len(counts)]], counts, 8 * group, 8, 128, 64, wide=wide)
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=max(counts), want_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
    side.synchronize()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
    for i in range(3):
        q.mul_(1.25)
        rows.copy_(dr.rows_of(dr.ways_of(dr.parents_of(counts, 70 + i)), rows.shape[1]))
        cache.lengths -= 3
        graph.replay()
        eager = pa.attention_kv8_tree(q, *cache.operands(pa), rows, **kw)
        assert pa.last_kernel() == kernel
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1]), i


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("kv_heads,dim,tokens,group", [(160, 128, 64, 2), (96, 128, 70, 4), (200, 64, 66, 1), (200, 64, 200, 2)])
def test_the_last_pages_of_a_cache_of_more_than_4_gib(pa, code, kv_heads, dim, tokens, group):  # noqa: F811
    """As the same pages of a small cache, bit for bit."""
    counts = [tokens, 3, tokens // 2]
    small = ref.Cache(code, [n + o for n, o in zip(counts, (300, 0, 130))], kv_heads, dim, 256, 31)
    q = queries(sum(counts), kv_heads * group, dim, torch.bfloat16, 32)
    ways = dr.ways_of(dr.parents_of(counts, 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    print("large", code, kv_heads, dim, counts, flush=True)
    expected = call(pa, WHOLE, q, small, rows, counts)
    ref.check_attention(expected[0], expected_of(q, small, ways), expected[1])
    first = 2 ** 32 // (kv_heads * 256 * dim) + 5
    large = types.SimpleNamespace(**vars(small))
    large.operands = types.MethodType(ref.Cache.operands, large)
    for name in ("k", "v"):
        x = torch.empty((first + small.k.shape[0], kv_heads, 256, dim), dtype=torch.uint8, device="cuda")
        x[first:] = getattr(small, name)
        s = torch.full((x.shape[0], kv_heads), 1.0, device="cuda")
        s[first:] = getattr(small, name + "_scale")
        setattr(large, name, x)
        setattr(large, name + "_scale", s)
    large.table = torch.where(small.table >= 0, small.table + first, small.table)
    got = call(pa, WHOLE, q, large, rows, counts)
    assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


@pytest.mark.parametrize("kv_heads,dim,tokens,group", [(160, 128, 64, 2), (64, 128, 70, 4), (200, 64, 66, 2), (100, 64, 200, 2)])
def test_places_at_the_end_of_the_longest_table(pa, kv_heads, dim, tokens, group):  # noqa: F811
    """2^31 - 2^16 tokens, a window over the last of them: as a sequence of those alone, bit for bit (whole: the same tiles of keys)."""
    short = ref.Cache("i8", [1024], kv_heads, dim, 256, 33)
    long = types.SimpleNamespace(**vars(short))
    long.operands = types.MethodType(ref.Cache.operands, long)
    blocks = (2 ** 31 - 2 ** 16) // 256
    long.table = torch.full((1, blocks), -1, dtype=torch.int32, device="cuda")
    long.table[0, -4:] = short.table[0, :4]
    long.lengths = torch.tensor([blocks * 256], dtype=torch.int32, device="cuda")
    q = queries(tokens, kv_heads * group, dim, torch.bfloat16, 34)
    ways = dr.ways_of(dr.parents_of([tokens], 6))
    rows = dr.rows_of(ways, -(-tokens // 64))
    print("places", kv_heads, dim, tokens, flush=True)
    expected = call(pa, WHOLE, q, short, rows, [tokens], window=220)
    ref.check_attention(expected[0], expected_of(q, short, ways, window=220), expected[1])
    got = call(pa, WHOLE, q, long, rows, [tokens], window=220)
    assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


def test_calls_on_two_streams_have_workspaces_of_their_own(pa):  # noqa: F811
    """Split calls on two streams and allocations on a third, nothing waited for in between: as the same calls one by one, bit for bit."""
    sides, work, tokens = [torch.cuda.Stream() for _ in range(2)], [], 32
    for seed in (41, 42):
        cache = widened(ref.Cache("e4m3", [5000, 500], 2, 128, 64, seed), 2 ** 20)
        q = queries(2 * tokens, 8, 128, torch.bfloat16, seed)
        rows = dr.rows_of(dr.ways_of(dr.parents_of([tokens] * 2, seed)), 1)
        need = pa.attention_kv8_tree_workspace_bytes(q, cache.k, cache.table, tokens)
        work.append((cache, q, rows, call(pa, CUT, q, cache, rows, [tokens] * 2)[0], need))
    got = [[torch.empty_like(q) for _ in range(20)] for _, q, _, _, _ in work]
    torch.cuda.synchronize()
    for i in range(20):
        for (cache, q, rows, _, need), side, outs in zip(work, sides, got):
            pa.attention_kv8_tree(q, *cache.operands(pa), rows, out=outs[i], stream=side)
            torch.empty(need, dtype=torch.uint8, device="cuda").fill_(0xFF)  # (the current stream's next owner of such a block)
    torch.cuda.synchronize()
    for (_, _, _, expected, _), outs in zip(work, got):
        for i, out in enumerate(outs):
            assert torch.equal(out, expected), i
