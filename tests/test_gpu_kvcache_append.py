"""The append to a cache held in 8 bits against its definition."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def append(pa, cache, k, v, counts, **kw):
    print("append", cache.code, counts[:4], cache.page, cache.dim, k.dtype, flush=True)
    pa.kvcache_append(k, v, *cache.operands(pa), cu_tokens=ref.starts(counts), max_tokens=max(counts), **kw)


def values(tokens, heads, dim, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(size * torch.randn((tokens, heads, dim), generator=g, device="cuda")).to(dtype) for _ in range(2)]


def nearest(codes, want, code):
    """Whether codes are nearest to `want` in units of their scale (f32 products before the rounding: 2^-22 of slack)."""
    got = ref.code_values(codes, code)
    unit = 1.0 if code == "i8" else torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -6))) - 3)
    return bool(((got - want).abs() <= 0.5 * unit * (1 + 2.0 ** -10) + 2.0 ** -22 * want.abs()).all())


def check(cache, before, k, v, counts):
    """Scales by their formula in f32, bit for bit, codes nearest in units of the scale that is there, everything else untouched."""
    for name, x in (("k", k), ("v", v)):
        codes, scales = getattr(cache, name), getattr(cache, name + "_scale")
        old_codes, old_scales = before[name], before[name + "_scale"]
        expected_same = torch.ones(codes.shape[:3], dtype=torch.bool, device="cuda")
        scales_same = torch.ones(scales.shape[0], dtype=torch.bool, device="cuda")
        at = 0
        for s, n in enumerate(counts):
            length, table = int(cache.lengths[s]), cache.table[s].tolist()
            start = length - n
            for b in range(start // cache.page, -(-length // cache.page) if n else 0):
                lo, hi, page = max(start, b * cache.page), min(length, (b + 1) * cache.page), table[b]
                older, rows = lo - b * cache.page, x[at + lo - start:at + hi - start].double().transpose(0, 1)
                unit = rows.abs().amax(dim=(1, 2)).float() * torch.tensor(1.0 / ref.LARGEST[cache.code], device="cuda")  # (both in f32)
                if older:
                    unit = torch.maximum(unit, old_scales[page])
                now = scales[page].double()
                assert torch.equal(scales[page], torch.where(unit < 2.0 ** -126, 0.0, unit)), (name, s, b)
                per = torch.where(now > 0, now, 1.0)[:, None, None]
                assert nearest(codes[page, :, older:older + hi - lo].contiguous(), rows / per, cache.code), (name, s, b)
                if older:
                    held = ref.code_values(old_codes[page, :, :older].contiguous(), cache.code) * old_scales[page].double()[:, None, None] / per
                    assert nearest(codes[page, :, :older].contiguous(), held, cache.code), (name, s, b)
                    expected_same[page, :, :older] = False
                expected_same[page, :, older:older + hi - lo] = False
                scales_same[page] = False
            at += n
        assert torch.equal(codes[expected_same], old_codes[expected_same])
        assert torch.equal(scales[scales_same].view(torch.int32), old_scales[scales_same].view(torch.int32))


def snapshot(cache):
    return {n: getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")}


def grown(code, olds, counts, heads, dim, page, seed, **kw):
    """A cache that holds `olds` tokens and whose lengths count the new ones too."""
    cache = ref.Cache(code, olds, heads, dim, page, seed, room=max(counts), **kw)
    cache.lengths = torch.tensor([o + n for o, n in zip(olds, counts)], dtype=torch.int32, device="cuda")
    return cache


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32), (80, 128), (8, 16), (512, 256)])
@pytest.mark.parametrize("counts", [[1] * 8, [130, 0, 1, 63, 64, 65, 17, 400]])
def test_against_the_definition(pa, code, dtype, dim, page, counts):  # noqa: F811
    olds = [0, 1, 15, 16, 63, 64, 100, 31]
    cache = grown(code, olds, counts, 3, dim, page, 2)
    k, v = values(sum(counts), 3, dim, dtype, 3)
    v = v * 0.01  # (keys' scales mostly grow, values' mostly stay)
    before = snapshot(cache)
    append(pa, cache, k, v, counts)
    check(cache, before, k, v, counts)
    again = snapshot(cache)
    append(pa, cache, k, v, counts)  # the same tokens once more: nothing changes
    for n, t in again.items():
        assert torch.equal(t.view(torch.uint8), getattr(cache, n).view(torch.uint8)), n


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_views_and_token_major_caches(pa, offset):  # noqa: F811
    olds, counts = [5, 70], [3, 40]
    cache = grown("e4m3", olds, counts, 4, 64, 32, 4, token_major=True)
    whole = torch.randn((43, 9, 80), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").bfloat16()
    k, v = whole[:, 1:5, offset:offset + 64], whole[:, 5:9, offset:offset + 64]
    before = snapshot(cache)
    append(pa, cache, k, v, counts)
    check(cache, before, k, v, counts)


def test_equal_shares_without_starts(pa):  # noqa: F811
    caches = [grown("i8", [9, 30], [4, 4], 2, 128, 16, 6) for _ in range(2)]
    k, v = values(8, 2, 128, torch.float16, 7)
    append(pa, caches[0], k, v, [4, 4])
    pa.kvcache_append(k, v, *caches[1].operands(pa))
    assert all(torch.equal(getattr(caches[0], n).view(torch.uint8), getattr(caches[1], n).view(torch.uint8)) for n in ("k", "v", "k_scale", "v_scale"))


def test_one_by_one_is_close_to_all_at_once(pa):  # noqa: F811
    """A page filled token by token is rounded again where its scale grows: every value within a scale's unit (int8) for each growth, at
    most as many as tokens, of what was appended; the scale itself is that of the whole page."""
    k, v = values(64, 2, 128, torch.bfloat16, 8)
    whole = grown("i8", [0], [64], 2, 128, 64, 9)
    append(pa, whole, k, v, [64])
    steps = grown("i8", [0], [64], 2, 128, 64, 9)
    for t in range(64):
        steps.lengths.fill_(t + 1)
        append(pa, steps, k[t:t + 1], v[t:t + 1], [1])
    page = int(steps.table[0, 0])
    assert torch.equal(steps.k_scale[page], whole.k_scale[int(whole.table[0, 0])])
    held = ref.code_values(steps.k[page].contiguous(), "i8")
    want = k.double().transpose(0, 1) / steps.k_scale[page].double()[:, None, None]
    growths = 8  # (a maximum over 64 tokens of 128 values is set anew 1 + 1/2 + ... + 1/64 = 4.7 times on average)
    assert float((held - want).abs().max()) <= 0.5 * (1 + growths)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_zeros_and_tiny_values(pa, code):  # noqa: F811
    cache = grown(code, [0, 0, 10], [20, 20, 4], 2, 64, 32, 10)
    k, v = values(44, 2, 64, torch.float32, 11)
    k[:20] = 0.0
    k[20:40] *= 1e-38 / 4
    before = snapshot(cache)
    append(pa, cache, k, v, [20, 20, 4])
    for s in range(2):
        page = int(cache.table[s, 0])
        assert bool((cache.k_scale[page] == 0).all()) and bool((ref.code_values(cache.k[page, :, :20].contiguous(), code) == 0).all())
    k[20:40] = 0.0
    check(cache, before, k, v, [20, 20, 4])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_values_that_are_no_numbers(pa, code, bad):  # noqa: F811
    """They make the scale of their page and head NaN, for good; the others are as ever."""
    olds, counts = [3, 40], [50, 50]
    cache, clean = (grown(code, olds, counts, 2, 64, 32, 12) for _ in range(2))
    k, v = values(100, 2, 64, torch.bfloat16, 13)
    append(pa, clean, k, v, counts)
    k[7, 1, 9] = bad  # sequence 0, place 10: its first page
    append(pa, cache, k, v, counts)
    page = int(cache.table[0, 0])
    assert math.isnan(float(cache.k_scale[page, 1])) and math.isfinite(float(cache.k_scale[page, 0]))
    assert torch.equal(cache.v_scale.view(torch.int32), clean.v_scale.view(torch.int32)) and torch.equal(cache.v, clean.v)
    other = torch.ones(cache.k.shape[:2], dtype=torch.bool, device="cuda")
    other[page, 1] = False
    assert torch.equal(cache.k[other], clean.k[other])
    q = torch.randn((2, 2, 64), device="cuda").bfloat16()
    out = pa.attention_kv8(q, *cache.operands(pa))
    assert bool(out[0, 1].isnan().all()) and not bool(out[0, 0].isnan().any()) and not bool(out[1].isnan().any())


def test_tokens_without_a_place_are_left_out(pa):  # noqa: F811
    """More new tokens than the length counts, a length beyond the table, table entries that are no pages: nothing outside is written."""
    cache = ref.Cache("i8", [16, 16, 16], 1, 64, 16, 14)
    before = snapshot(cache)
    k, v = values(60, 1, 64, torch.float32, 15)
    cache.lengths = torch.tensor([5, 16 * cache.table.shape[1] + 9, 24], dtype=torch.int32, device="cuda")
    append(pa, cache, k, v, [20, 20, 20])
    first = int(cache.table[0, 0])
    assert nearest(cache.k[first, 0, :5], k[15:20, 0].double() / cache.k_scale[first].double(), "i8")
    assert torch.equal(cache.k[first, 0, 5:], before["k"][first, 0, 5:])
    second, third = int(cache.table[1, 0]), int(cache.table[2, 0])
    changed = {int(p) for p in (cache.k != before["k"]).any(dim=3).any(dim=2).any(dim=1).nonzero()}
    assert changed <= {first, second, third}, (changed, first, second, third)
    assert nearest(cache.k[third, 0, 4:], k[40:52, 0].double() / cache.k_scale[third].double(), "i8")


def test_captured(pa):  # noqa: F811
    cache, eager = (grown("e4m3", [10, 30], [1, 1], 2, 128, 32, 16) for _ in range(2))
    k, v = values(2, 2, 128, torch.bfloat16, 17)
    graph = torch.cuda.CUDAGraph()
    lengths = cache.lengths
    with torch.cuda.graph(graph):
        pa.kvcache_append(k, v, *cache.operands(pa))
    for i in range(4):
        graph.replay()
        pa.kvcache_append(k, v, *eager.operands(pa))
        assert all(torch.equal(getattr(cache, n).view(torch.uint8), getattr(eager, n).view(torch.uint8)) for n in ("k", "v", "k_scale", "v_scale")), i
        k.mul_(1.3)
        lengths.add_(1)
        eager.lengths.add_(1)
    del graph
