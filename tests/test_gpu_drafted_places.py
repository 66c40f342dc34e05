"""The operators around drafted trees where offsets and places pass 32 bits or nearly, and on streams that are not the current one."""
import types

import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def step(pa, cache, counts, heads, seed, window=0):  # noqa: F811
    """Append, attention and keep of a tree: every result."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda n: torch.randn((sum(counts), n, cache.dim), generator=g, device="cuda").bfloat16()  # noqa: E731
    q, k, v = draw(heads), draw(cache.kv_heads), draw(cache.kv_heads)
    cu, most = ref.starts(counts), max(counts)
    parents = dr.parents_of(counts, seed)
    tree = pa.draft_tree(dr.flat(parents), len(counts), cu, most)
    table = pa.rope_table(4096, 64)
    positions = torch.arange(sum(counts), dtype=torch.int32, device="cuda")
    turned = pa.kvcache_append_rope(q, k, v, *cache.operands(pa), table, positions, cu_tokens=cu, max_tokens=most)
    out, lse = pa.attention_kv8_tree(turned, *cache.operands(pa), tree, cu_tokens=cu, max_tokens=most, window=window, want_lse=True)
    kept = torch.tensor([[n // 3, n // 2, n - 1] for n in counts], dtype=torch.int32, device="cuda")
    lengths = pa.kvcache_keep(kept, *cache.operands(pa), cu_tokens=cu, max_tokens=most)
    return turned, out, lse, lengths


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("kv_heads,dim,counts", [(8, 128, [7, 70, 5]), (8, 256, [40, 9, 3]), (16, 64, [130, 3, 60])])
def test_caches_of_more_than_4_gib(pa, code, kv_heads, dim, counts):  # noqa: F811
    """The last pages of a large cache as the same pages of a small one, bit for bit."""
    small = ref.Cache(code, [n + o for n, o in zip(counts, (700, 250, 1000))], kv_heads, dim, 256, 31)
    pages = small.k.shape[0]
    first = 2 ** 32 // (kv_heads * 256 * dim) + 5
    large = types.SimpleNamespace(**vars(small))
    for name in ("k", "v"):
        x = torch.empty((first + pages, kv_heads, 256, dim), dtype=torch.uint8, device="cuda")
        x[first:] = getattr(small, name)
        s = torch.full((first + pages, kv_heads), 1.0, device="cuda")
        s[first:] = getattr(small, name + "_scale")
        setattr(large, name, x)
        setattr(large, name + "_scale", s)
    large.table = torch.where(small.table >= 0, small.table + first, small.table)
    large.operands = types.MethodType(ref.Cache.operands, large)
    print("large", code, kv_heads, dim, counts, flush=True)
    expected = step(pa, small, counts, 2 * kv_heads, 32)
    for got, want in zip(step(pa, large, counts, 2 * kv_heads, 32), expected):
        assert torch.equal(got, want)
    for name in ("k", "v", "k_scale", "v_scale"):
        got, want = getattr(large, name)[first:], getattr(small, name)
        assert torch.equal(got.view(torch.uint8) if got.dtype == torch.uint8 else got.view(torch.int32), want if want.dtype == torch.uint8 else want.view(torch.int32))


@pytest.mark.parametrize("dim,tokens", [(64, 5), (128, 5), (256, 5), (64, 120), (128, 120), (256, 120), (72, 20)])
def test_places_at_the_end_of_the_longest_table(pa, dim, tokens):  # noqa: F811
    """2^31 - 2^16 tokens, a window over the last of them: as a sequence of those alone."""
    short = ref.Cache("i8", [1024], 2, dim, 256, 33)
    long = types.SimpleNamespace(**{k: v.clone() if torch.is_tensor(v) else v for k, v in vars(short).items()})
    long.operands = types.MethodType(ref.Cache.operands, long)
    blocks = (2 ** 31 - 2 ** 16) // 256
    long.table = torch.full((1, blocks), -1, dtype=torch.int32, device="cuda")
    long.table[0, -4:] = short.table[0, :4]
    long.lengths = torch.tensor([blocks * 256], dtype=torch.int32, device="cuda")
    print("places", dim, tokens, flush=True)
    turned, out, lse, lengths = step(pa, long, [tokens], 8, 34, window=300)
    expected, expected_out, expected_lse, expected_lengths = step(pa, short, [tokens], 8, 34, window=300)
    assert torch.equal(turned, expected) and torch.equal(lengths - expected_lengths, long.lengths - 1024)
    for name in ("k", "v"):
        assert torch.equal(getattr(long, name), getattr(short, name))
        assert torch.equal(getattr(long, name + "_scale").view(torch.int32), getattr(short, name + "_scale").view(torch.int32))  # (bits: spare pages' are NaN)
    # (the keys may be cut elsewhere.  Each result is off by the rounding of its weights to f16 and its own to bf16, 2^-11 and 2^-8; values are below 6.)
    off = (out.float() - expected_out.float()).abs()
    assert bool((off <= 2 * (2.0 ** -8 * expected_out.float().abs() * (1 + 2.0 ** -7) + 2.0 ** -11 * 6)).all()) and bool(((lse - expected_lse).abs() <= 2.0 ** -10).all())


@pytest.mark.parametrize("tokens", [1, 12, 70])
def test_calls_on_two_streams_have_workspaces_of_their_own(pa, tokens):  # noqa: F811
    """Split calls on two streams and allocations on a third, nothing waited for in between: as the same calls one by one, bit for bit."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for seed in (41, 42):
        cache = ref.Cache("e4m3", [9000, 500], 2, 128, 64, seed)
        q = torch.randn((2 * tokens, 16, 128), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
        ways = dr.ways_of(dr.parents_of([tokens] * 2, seed))
        rows = dr.rows_of(ways, -(-tokens // 64))
        need = pa.attention_kv8_tree_workspace_bytes(q, cache.k, cache.table, tokens)
        assert need > 0
        out, lse = pa.attention_kv8_tree(q, *cache.operands(pa), rows, want_lse=True)
        ref.check_attention(out, dr.attention(q, cache, ways), lse)
        work.append((cache, q, rows, out, need))
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
