"""Keeping a path of drafted tokens in a cache held in 8 bits, against its definition."""
import math
import random

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_kvcache_append import nearest, snapshot
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def paths(counts, most, seed):
    """The way to some token of a tree of each, as far as `most`."""
    rng = random.Random(seed)
    kept = []
    for ways in dr.ways_of(dr.parents_of(counts, seed, 0 if seed % 2 else 3)):
        kept.append(sorted(ways[rng.randrange(len(ways))])[:most] if ways else [])
    return kept


def listed(kept, most, fill=-1):
    return torch.tensor([mine + [fill] * (most - len(mine)) for mine in kept], dtype=torch.int32, device="cuda").view(len(kept), most)


def check(cache, before, counts, kept, lengths):
    """Scales by their formula in f32, bit for bit; codes copied within a page, nearest where a scale is another; everything else untouched."""
    want_lengths = []
    for name in ("k", "v"):
        codes, scales, old_codes, old_scales = getattr(cache, name), getattr(cache, name + "_scale"), before[name], before[name + "_scale"]
        codes_same = torch.ones(codes.shape[:3], dtype=torch.bool, device="cuda")
        scales_same = torch.ones(scales.shape[0], dtype=torch.bool, device="cuda")
        for s, (n, mine) in enumerate(zip(counts, kept)):
            start, table = int(cache.lengths[s]) - n, cache.table[s].tolist()
            want_lengths.append(start + len(mine))
            for b in sorted({(start + r) // cache.page for r in range(len(mine))}):
                page, here = table[b], [r for r in range(len(mine)) if (start + r) // cache.page == b]
                unit, comes = old_scales[page].clone(), False
                for r in here:
                    sb, slot = divmod(start + mine[r], cache.page)
                    if sb != b:
                        size = ref.code_values(old_codes[table[sb], :, slot].contiguous(), cache.code).float().abs().amax(dim=1) * old_scales[table[sb]]
                        unit, comes = torch.maximum(unit, size * torch.tensor(1.0 / ref.LARGEST[cache.code], device="cuda")), True
                if comes:
                    unit = torch.where(unit < 2.0 ** -126, 0.0, unit)
                    assert torch.equal(scales[page], unit), (name, s, b)
                    scales_same[page] = False
                now = scales[page].double()
                per = torch.where(now > 0, now, 1.0)[:, None]
                older = max(0, start - b * cache.page)
                held = [(slot, page, slot) for slot in range(older)] + [((start + r) % cache.page, table[(start + mine[r]) // cache.page], (start + mine[r]) % cache.page)
                                                                         for r in here]
                for slot, source, source_slot in held:
                    was = old_codes[source, :, source_slot].contiguous()
                    got = codes[page, :, slot].contiguous()
                    alike = old_scales[source] == scales[page]
                    assert torch.equal(got[alike], was[alike]), (name, s, b, slot)
                    value = ref.code_values(was, cache.code) * old_scales[source].double()[:, None] / per
                    assert nearest(got, value, cache.code), (name, s, b, slot)
                    codes_same[page, :, slot] = False
        assert torch.equal(codes[codes_same], old_codes[codes_same])
        assert torch.equal(scales[scales_same].view(torch.int32), old_scales[scales_same].view(torch.int32))
    assert lengths.tolist() == want_lengths[:len(counts)]


def run(pa, code, olds, counts, kept, most, heads, dim, page, seed, factor=1.0, **kw):
    cache = ref.Cache(code, [o + n for o, n in zip(olds, counts)], heads, dim, page, seed, **kw)
    if factor != 1.0:  # (every second page's scales)
        for table in cache.table.tolist():
            for p in table[1::2]:
                if p >= 0:
                    cache.k_scale[p] *= factor
                    cache.v_scale[p] /= factor
    print("keep", code, olds[:4], counts[:4], [len(m) for m in kept][:4], heads, dim, page, flush=True)
    before = snapshot(cache)
    lengths = pa.kvcache_keep(listed(kept, most), *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=max(counts))
    check(cache, before, counts, kept, lengths)
    return cache, lengths


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32), (80, 128), (8, 16), (512, 256), (72, 16)])
@pytest.mark.parametrize("factor", [1.0, 3.7, 2.0 ** 20])
def test_paths_of_trees(pa, code, dim, page, factor):  # noqa: F811
    olds, counts = [0, 1, 15, 16, 63, 64, 100, 31], [130, 0, 1, 63, 64, 200, 17, 256]
    for seed in (1, 2):
        run(pa, code, olds, counts, paths(counts, 12, seed), 12, 3, dim, page, seed, factor)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_paths_of_any_length(pa, code, page, dim):  # noqa: F811
    """None, all of them, every second one, the last ones, which come from pages far behind."""
    olds, counts = [5, 70, 16, 0, 31], [256, 256, 100, 256, 200]
    kept = [list(range(256)), list(range(0, 256, 2)), [], list(range(156, 256)), sorted(random.Random(3).sample(range(200), 150))]
    run(pa, code, olds, counts, kept, 256, 2, dim, page, 4, 2.5, token_major=True)


def test_lists_end_where_they_are_out_of_order(pa):  # noqa: F811
    counts = [20] * 6
    rows = [[0, 3, 3, 5], [2, 1, 7, 9], [20, 1, 2, 3], [4, 19, 20, 21], [-5, 3, 4, 5], [0, 5, 2 ** 31 - 1, -2 ** 31]]
    kept = [[0, 3], [2], [], [4, 19], [], [0, 5]]
    cache = ref.Cache("i8", [30] * 6, 2, 64, 16, 5)
    before = snapshot(cache)
    lengths = pa.kvcache_keep(torch.tensor(rows, dtype=torch.int32, device="cuda"), *cache.operands(pa), max_tokens=20)
    check(cache, before, counts, kept, lengths)
    lengths = pa.kvcache_keep(torch.empty((6, 0), dtype=torch.int32, device="cuda"), *cache.operands(pa), max_tokens=20)
    assert lengths.tolist() == [10] * 6


def test_sequences_without_room_for_their_tokens_are_left_alone(pa):  # noqa: F811
    cache = ref.Cache("e4m3", [30, 30, 30], 2, 64, 16, 6)
    cache.lengths = torch.tensor([3, 200, -4], dtype=torch.int32, device="cuda")
    before = snapshot(cache)
    lengths = pa.kvcache_keep(listed([[1, 2]] * 3, 4), *cache.operands(pa), max_tokens=5)
    assert lengths.tolist() == [3, 200, 0]
    for n, t in before.items():
        assert torch.equal(getattr(cache, n).view(torch.uint8), t.view(torch.uint8))


def test_pages_that_are_none_and_scales_that_are_no_numbers(pa):  # noqa: F811
    """A token that comes from a page that the table does not name, or whose scale is NaN: the scale of the page that it comes to is NaN; a page that is
    none takes nothing; a page that nothing comes into keeps its scale."""
    olds, counts = [14] * 4, [40] * 4
    kept = [[0, 1, 20, 39]] * 4  # places 14, 15 | 16, 17 from pages 2 and 3
    cache = ref.Cache("i8", [54] * 4, 2, 64, 16, 7)
    before = snapshot(cache)
    pages = cache.table.clone()
    cache.table[0, 3] = -1
    cache.v_scale[pages[1, 2].long(), 1] = math.nan
    cache.table[2, 1] = 1 << 20
    nan_before = cache.k_scale[pages[3, 0].long(), 0] = math.nan
    assert math.isnan(nan_before)
    pa.kvcache_keep(listed(kept, 4), *cache.operands(pa), max_tokens=40)
    to = pages[:, 1].long()
    assert bool(cache.k_scale[to[0]].isnan().all()) and bool(cache.v_scale[to[0]].isnan().all())
    assert cache.v_scale[to[1]].isnan().tolist() == [False, True] and not bool(cache.k_scale[to[1]].isnan().any())
    for n in ("k", "v"):
        assert torch.equal(getattr(cache, n)[to[2]], before[n][to[2]]) and torch.equal(getattr(cache, n + "_scale")[to[2]], before[n + "_scale"][to[2]])
        assert torch.equal(getattr(cache, n)[pages[3, 0].long()], before[n][pages[3, 0].long()])
    assert cache.k_scale[pages[3, 0].long()].isnan().tolist() == [True, False]
    assert not bool(cache.k_scale[to[3]].isnan().any())


def test_zero_scales(pa):  # noqa: F811
    """A page of zeros takes tokens of another, and a page takes tokens of one of zeros."""
    for zero in (1, 2):
        cache = ref.Cache("e4m3", [54], 2, 64, 16, 8)
        page = cache.table[0, zero].long()
        cache.k_scale[page], cache.v_scale[page] = 0.0, 0.0
        cache.k[page, :, :], cache.v[page, :, :] = 0, 0
        before = snapshot(cache)
        lengths = pa.kvcache_keep(listed([[0, 1, 20, 39]], 4), *cache.operands(pa), max_tokens=40)
        check(cache, before, [40], [[0, 1, 20, 39]], lengths)


def test_captured_on_another_stream_and_into_a_given_tensor(pa):  # noqa: F811
    counts = [50] * 4
    caches = [ref.Cache("i8", [90, 64, 50, 127], 2, 128, 16, 9) for _ in range(2)]
    kept = listed(paths(counts, 8, 1), 8)
    out = torch.full((4,), 77, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pa.kvcache_keep(kept, *caches[0].operands(pa), max_tokens=50, out=out)
    assert got is out
    side = torch.cuda.Stream()
    for i in range(4):
        kept.copy_(listed(paths(counts, 8, 30 + i), 8))
        torch.cuda.synchronize()
        graph.replay()
        there = torch.empty_like(out)
        torch.cuda.synchronize()
        pa.kvcache_keep(kept, *caches[1].operands(pa), max_tokens=50, out=there, stream=side)
        side.synchronize()
        assert torch.equal(out, there)
        for n in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(caches[0], n).view(torch.uint8), getattr(caches[1], n).view(torch.uint8)), (i, n)


def test_what_is_kept_is_what_attention_then_sees(pa):  # noqa: F811
    """Attention over the kept cache: as over the drafted one along the path, values within a code's rounding where tokens changed their page: half a step of
    int8 a scale that is at most twice the other pages', 1 / 127 of the largest."""
    counts, olds = [60], [100]
    kept = paths(counts, 9, 4)
    cache = ref.Cache("i8", [160], 2, 128, 16, 10)
    q = torch.randn((60, 8, 128), generator=torch.Generator(device="cuda").manual_seed(11), device="cuda").bfloat16()
    last = kept[0][-1]
    ways = [[set(kept[0]) for _ in range(60)]]
    drafted = pa.attention_kv8_tree(q, *cache.operands(pa), dr.rows_of(ways, 1))[last]
    cache.lengths = pa.kvcache_keep(listed(kept, 9), *cache.operands(pa), max_tokens=60)
    after = pa.attention_kv8(q[last:last + 1].contiguous(), *cache.operands(pa))[0]
    size = max(float(x[0].abs().max()) for x in (cache.kd, cache.vd))
    assert float((after.float() - drafted.float()).abs().max()) <= 4 * size / 127
