"""The append with rotation on the way: bit for bit what the rotation in f32 and the append of its results give, and against the definition in 64 bits."""
import math

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_kvcache_append import check as check_append
from test_gpu_kvcache_append import grown, snapshot
from test_gpu_parity import pa  # noqa: F401
from test_gpu_rope import check as check_rope

pytestmark = pytest.mark.gpu
NAMES = ("k", "v", "k_scale", "v_scale")


def fused(tokens, heads, kv_heads, dim, dtype, seed, offset=0):
    """Queries, keys and values side by side, as a product leaves them; rows that start on any element."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = torch.randn((tokens, heads + 2 * kv_heads, dim + 16), generator=g, device="cuda").to(dtype)[..., offset:offset + dim]
    return whole[:, :heads], whole[:, heads:heads + kv_heads], whole[:, heads + kv_heads:] * 0.25


def two_calls(pa, cache, q, k, v, counts, table, positions, interleaved):
    """rope() and kvcache_append(), keys in f32 in between."""
    turned = pa.rope(q, table, positions, interleaved=interleaved)
    keys = pa.rope(k.float(), table, positions, interleaved=interleaved)
    pa.kvcache_append(keys, v.float(), *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=max(counts))
    return turned


def same(a, b):
    for n in NAMES:
        assert torch.equal(getattr(a, n).view(torch.uint8), getattr(b, n).view(torch.uint8)), n


def places(olds, counts):
    return torch.tensor([o + i for o, n in zip(olds, counts) for i in range(n)], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,page", [(64, 64, 16), (128, 128, 64), (256, 64, 32), (80, 80, 128), (80, 32, 16), (96, 24, 32), (8, 2, 16), (512, 512, 256), (72, 16, 64), (64, 48, 256)])
def test_as_the_two_calls(pa, code, dtype, interleaved, dim, rot, page):  # noqa: F811
    olds, counts = [0, 1, 15, 16, 63, 64, 100, 31], [130, 0, 1, 63, 64, 65, 17, 200]
    table = pa.rope_table(300, rot)
    q, k, v = fused(sum(counts), 5, 3, dim, dtype, dim + rot)
    caches = [grown(code, olds, counts, 3, dim, page, 2) for _ in range(2)]
    expected = two_calls(pa, caches[0], q, k, v, counts, table, places(olds, counts), interleaved)
    got = pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table, interleaved=interleaved, cu_tokens=ref.starts(counts), max_tokens=max(counts))
    assert pa.last_kernel() == "kvcache_append_rope"
    assert torch.equal(got, expected)
    same(*caches)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (72, 8), (7, 7), (64, 2), (0, 3)])
@pytest.mark.parametrize("counts", [[1] * 7, [4] * 3, [1, 0, 2, 1, 33]])
def test_steps_of_few_tokens(pa, code, heads, kv_heads, counts):  # noqa: F811
    olds = [0, 70, 15, 16, 127, 3, 64][:len(counts)]
    table = pa.rope_table(300, 128)
    q, k, v = fused(sum(counts), max(heads, 1), kv_heads, 128, torch.bfloat16, heads)
    caches = [grown(code, olds, counts, kv_heads, 128, 64, 5) for _ in range(2)]
    expected = two_calls(pa, caches[0], q, k, v, counts, table, places(olds, counts), False)
    kw = dict(cu_tokens=ref.starts(counts), max_tokens=max(counts)) if len(set(counts)) > 1 else {}
    got = pa.kvcache_append_rope(q if heads else None, k, v, *caches[1].operands(pa), table, **kw)
    assert (got is None) if not heads else torch.equal(got, expected)
    same(*caches)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_the_definition(pa, dtype, interleaved):  # noqa: F811
    """Queries as rope's.  Keys: what the cache holds after appending keys that were turned in 64 bits and rounded to f32, of which a rotated element
    in f32 is off by two products' and a sum's rounding: scales within 2^-22, codes within one of the nearest (half a step and what is off)."""
    olds, counts = [0, 17, 40], [50, 3, 90]
    table = pa.rope_table(300, 64)
    q, k, v = fused(143, 4, 2, 64, dtype, 3)
    positions = places(olds, counts)
    cache = grown("e4m3", olds, counts, 2, 64, 32, 6)
    before = snapshot(cache)
    got = pa.kvcache_append_rope(q, k, v, *cache.operands(pa), table, interleaved=interleaved, cu_tokens=ref.starts(counts), max_tokens=90)
    check_rope(got, q, table, positions, interleaved, False)
    turned = pa.rope(k.float(), table, positions, interleaved=interleaved)
    check_rope(turned, k.float(), table, positions, interleaved, False)
    check_append(cache, before, turned, v.float(), counts)


@pytest.mark.parametrize("counts", [[24] * 5, [1, 0, 256, 33, 100]])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 20])
def test_positions_of_trees(pa, counts, interleaved, rot):  # noqa: F811
    """A drafted token stands behind those that it sees; bits behind a sequence's last token are not counted."""
    olds = [5, 0, 100, 16, 47]
    parents = dr.parents_of(counts, 7)
    ways = dr.ways_of(parents)
    depth = torch.tensor([o + len(w) - 1 for o, mine in zip(olds, ways) for w in mine], dtype=torch.int32, device="cuda")
    words = -(-max(counts) // 64)
    rows = dr.rows_of([[w | set(range(len(mine), 64 * words)) for w in mine] for mine in ways], words)
    table = pa.rope_table(400, rot)
    q, k, v = fused(sum(counts), 6, 2, 64, torch.bfloat16, 8)
    kw = dict(interleaved=interleaved, cu_tokens=ref.starts(counts), max_tokens=max(counts))
    caches = [grown("i8", olds, counts, 2, 64, 16, 9) for _ in range(3)]
    expected = two_calls(pa, caches[0], q, k, v, counts, table, depth, interleaved)
    assert torch.equal(pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table, tree=rows, **kw), expected)
    same(*caches[:2])
    assert torch.equal(pa.kvcache_append_rope(q, k, v, *caches[2].operands(pa), table, positions=depth, **kw), expected)
    same(*caches[1:])


def test_rows_of_bits_that_are_no_trees(pa):  # noqa: F811
    """An empty row stands where its sequence's older tokens end, as one that sees itself alone does; bits of later tokens count."""
    sets = [[set(), {1}, {0, 1, 2, 3}, {0, 2}, {4, 3}]]
    q, k, v = fused(5, 2, 2, 64, torch.float32, 11)
    table = pa.rope_table(60, 64)
    cache = grown("i8", [20], [5], 2, 64, 16, 12)
    got = pa.kvcache_append_rope(q, k, v, *cache.operands(pa), table, tree=dr.rows_of(sets, 1))
    assert torch.equal(got, pa.rope(q, table, torch.tensor([20, 20, 23, 22, 21], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 40])
def test_views_token_major_caches_and_in_place(pa, offset, interleaved, rot):  # noqa: F811
    olds, counts = [5, 70], [3, 40]
    table = pa.rope_table(200, rot)
    g = torch.Generator(device="cuda").manual_seed(5)
    whole = torch.randn((43, 13, 80), generator=g, device="cuda").bfloat16()
    q, k, v = whole[:, :5, offset:offset + 64], whole[:, 5:9, offset:offset + 64], whole[:, 9:, offset:offset + 64]
    caches = [grown("e4m3", olds, counts, 4, 64, 32, 4, token_major=True) for _ in range(2)]
    expected = two_calls(pa, caches[0], q, k, v, counts, table, places(olds, counts), interleaved)
    kept = whole.clone()
    got = pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table, interleaved=interleaved, cu_tokens=ref.starts(counts), max_tokens=40, out=q)
    assert got is q and torch.equal(q, expected)
    kept[:, :5, offset:offset + 64] = expected
    assert torch.equal(whole, kept)  # (nothing beside the result was written)
    same(*caches)


def test_positions_that_the_table_does_not_have(pa):  # noqa: F811
    """NaN queries, NaN key scales of the pages that such tokens come to; values and other pages as ever."""
    q, k, v = fused(4, 3, 2, 64, torch.bfloat16, 13)
    table = pa.rope_table(50, 32)
    positions = torch.tensor([7, 50, -1, 49], dtype=torch.int32, device="cuda")
    caches = [grown("i8", [3, 20, 33, 0], [1] * 4, 2, 64, 16, 14) for _ in range(2)]
    expected = two_calls(pa, caches[0], q, k, v, [1] * 4, table, positions, False)
    got = pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table, positions=positions)
    assert bool(got[1:3, :, :32].isnan().all()) and torch.equal(got[1:3, :, 32:], q[1:3, :, 32:]) and torch.equal(got[[0, 3]], expected[[0, 3]])
    assert bool(caches[1].k_scale[caches[1].table[1, 1].long()].isnan().all()) and not bool(caches[1].v_scale[caches[1].table[1, 1].long()].isnan().any())
    for n in ("k", "v"):
        assert torch.equal(getattr(caches[0], n), getattr(caches[1], n))
        assert torch.equal(getattr(caches[0], n + "_scale").nan_to_num(-1.0), getattr(caches[1], n + "_scale").nan_to_num(-1.0))


def test_tokens_without_a_place_and_pages_that_are_none(pa):  # noqa: F811
    """Fewer tokens than were given, more than the table holds, entries that name no page: left out as in an append; queries are turned all the same."""
    q, k, v = fused(30, 2, 2, 64, torch.float32, 15)
    table = pa.rope_table(200, 64)
    for lengths in ([4, 60], [48, 16], [0, -7], [130, 200]):
        caches = [grown("e4m3", [0, 5], [20, 10], 2, 64, 16, 16) for _ in range(2)]
        for c in caches:
            c.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            c.table[1, 0] = 1 << 20
        counts = [20, 10]
        positions = places([max(n, 0) - c for n, c in zip(lengths, counts)], counts)
        expected = two_calls(pa, caches[0], q, k, v, counts, table, positions, False)
        got = pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table, cu_tokens=ref.starts(counts), max_tokens=20)
        assert torch.equal(got.nan_to_num(7.0), expected.nan_to_num(7.0))
        for n in NAMES:
            a, b = (getattr(c, n) for c in caches)
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) if a.is_floating_point() else torch.equal(a, b), (lengths, n)


@pytest.mark.parametrize("sequences", [1, 2, 63, 64, 65, 130, 4096, 4097, 5000])
def test_any_number_of_sequences_and_loose_bounds(pa, sequences):  # noqa: F811
    """Ragged batches, sequences without tokens among them, behind the first rows and before the last of the batch, max_tokens up to all rows: queries as rope's at
    each token's place, caches as with the bound that is the most."""
    g = torch.Generator().manual_seed(sequences)
    counts = torch.randint(0, 4, (sequences,), generator=g, dtype=torch.int32)
    counts[torch.rand(sequences, generator=g) < 0.3] = 0
    counts[sequences // 2] = 9
    olds = torch.randint(0, 20, (sequences,), generator=g, dtype=torch.int32)
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), counts.cumsum(0, dtype=torch.int32)]) + 3
    used, rows = int(counts.sum()), int(counts.sum()) + 8
    owner = torch.repeat_interleave(torch.arange(sequences), counts.long())
    positions = torch.zeros(rows, dtype=torch.int32)
    positions[3:3 + used] = olds[owner] + torch.arange(used, dtype=torch.int32) - (cu[:-1] - 3)[owner]
    q, k, v = fused(rows, 6, 2, 64, torch.bfloat16, 19)
    table, lengths = pa.rope_table(64, 64), (olds + counts).cuda()
    expected = pa.rope(q, table, positions.cuda())
    results = []
    for most in (9, 2 * used, rows + 1000):
        cache = [torch.zeros((2 * sequences, 2, 16, 64), dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.zeros((2 * sequences, 2), device="cuda") for _ in range(2)]
        blocks = torch.arange(2 * sequences, dtype=torch.int32, device="cuda").view(sequences, 2)
        out = torch.full((rows, 6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        pa.kvcache_append_rope(q, k, v, *cache, blocks, lengths, pa.I8, table, cu_tokens=cu.cuda(), max_tokens=most, out=out)
        assert torch.equal(out[3:3 + used], expected[3:3 + used]) and bool((out[:3] == 7.0).all()) and bool((out[3 + used:] == 7.0).all())
        results.append(cache)
    assert bool((results[0][2] > 0).any())
    for cache in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(cache, results[0]))


@pytest.mark.parametrize("tree", [False, True])
def test_padded_batches(pa, tree):  # noqa: F811
    """Rows that no sequence has are neither read nor written."""
    counts, olds = [3, 0, 40], [30, 20, 50]
    q, k, v = fused(43, 4, 2, 64, torch.bfloat16, 17)
    table = pa.rope_table(200, 64)
    rows = dr.rows_of(dr.ways_of(dr.parents_of(counts, 3)), 1)
    caches = [grown("i8", olds, counts, 2, 64, 16, 18) for _ in range(2)]
    expected = pa.kvcache_append_rope(q, k, v, *caches[0].operands(pa), table, tree=rows if tree else None, cu_tokens=ref.starts(counts), max_tokens=40)
    wide = [torch.full((60, x.shape[1], 64), math.nan, dtype=torch.bfloat16, device="cuda") for x in (q, k, v)]
    for to, x in zip(wide, (q, k, v)):
        to[5:48] = x
    wide_rows = torch.full((60, 1), -1, dtype=torch.int64, device="cuda")
    wide_rows[5:48] = rows
    out = torch.full_like(wide[0], 7.0)
    pa.kvcache_append_rope(*wide, *caches[1].operands(pa), table, tree=wide_rows if tree else None, cu_tokens=ref.starts(counts) + 5, max_tokens=40, out=out)
    assert torch.equal(out[5:48], expected) and bool((out[:5] == 7.0).all()) and bool((out[48:] == 7.0).all())
    same(*caches)
    # beyond max_tokens: the first ones of each sequence alone
    out.fill_(7.0)
    pa.kvcache_append_rope(*wide, *caches[1].operands(pa), table, tree=wide_rows if tree else None, cu_tokens=ref.starts(counts) + 5, max_tokens=20, out=out)
    assert bool((out[5 + 3 + 20:] == 7.0).all()) and not bool((out[5:28] == 7.0).all(dim=(1, 2)).any())


def test_captured_and_on_another_stream(pa):  # noqa: F811
    q, k, v = fused(8, 16, 4, 128, torch.bfloat16, 19)
    table = pa.rope_table(500, 128)
    caches = [grown("e4m3", [100, 47], [0, 0], 4, 128, 32, 20) for _ in range(3)]
    for c in caches:  # (room for the tokens of all replays)
        c.table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
        c.k, c.v = (torch.zeros((64, 4, 32, 128), dtype=torch.uint8, device="cuda") for _ in range(2))
        c.k_scale, c.v_scale = (torch.zeros((64, 4), device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pa.kvcache_append_rope(q, k, v, *caches[0].operands(pa), table, out=out)
    for c in caches:
        for n in NAMES:
            getattr(c, n).zero_()
    side = torch.cuda.Stream()
    for i in range(4):
        for c in caches:
            c.lengths += 4
        graph.replay()
        eager = pa.kvcache_append_rope(q, k, v, *caches[1].operands(pa), table)
        assert torch.equal(out, eager), i
        same(caches[0], caches[1])
        other = torch.empty_like(q)
        torch.cuda.synchronize()
        pa.kvcache_append_rope(q, k, v, *caches[2].operands(pa), table, stream=side, out=other)
        side.synchronize()
        assert torch.equal(other, eager)
        same(caches[1], caches[2])
        q.mul_(0.75), k.mul_(1.5)
