"""The operators around drafted trees together: prompts in chunks, then trees of tokens of which one path is kept."""
import os
import sys

import pytest
import torch

from test_gpu_parity import pa  # noqa: F401

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import attention_layer as al  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,dim,error", [("E4M3", 128, 0.06), ("E4M3", 64, 0.06), ("I8", 128, 0.02), ("I8", 256, 0.02)])
@pytest.mark.parametrize("page", [16, 64])
def test_a_layer_serves_trees(pa, code, dim, error, page):  # noqa: F811
    """The relative error of a result is that of its inputs: E4M3 0.026, int8 0.0096 of keys and values each, as for prompts and steps; a token that changes its
    page is rounded once more, which adds as much again in squares: at most 0.052 and 0.0192 if all of them did."""
    layer = al.AttentionLayer(pa, width=512, heads=8, kv_heads=2, head_dim=dim, sequences=3, longest=400, page_size=page, code_type=getattr(pa, code))
    g = torch.Generator(device="cuda").manual_seed(2)
    prompts = [torch.randn((n, 512), generator=g, device="cuda").bfloat16() for n in (300, 171, 240)]
    outs = al.serve_drafted(layer, prompts, known=150, chunk=96, drafted=20)
    assert [o.shape for o in outs] == [p.shape for p in prompts]
    assert al.relative_error(layer, prompts, outs) < error


def test_a_step_allocates_nothing_beside_its_results(pa):  # noqa: F811
    """With out and a workspace given, the four calls allocate no device memory, in torch or behind its back."""
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.zeros((64, 4, 64, 128), dtype=torch.int8, device="cuda") for _ in range(2))
    k_scale, v_scale = (torch.zeros((64, 4), device="cuda") for _ in range(2))
    block_table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    lengths, after = torch.tensor([2048, 100], dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    turns = pa.rope_table(2048, 128)
    for tokens in (7, 70):
        x = torch.randn((2 * tokens, 24, 128), generator=g, device="cuda").bfloat16()
        parents = torch.arange(-1, tokens - 1, dtype=torch.int32, device="cuda").repeat(2)
        tree = torch.empty((2 * tokens, 2), dtype=torch.int64, device="cuda")
        kept = torch.tensor([[0, 1, 2, -1], [0, -1, -1, -1]], dtype=torch.int32, device="cuda")
        out = torch.empty((2 * tokens, 16, 128), dtype=torch.bfloat16, device="cuda")
        cache = (k, v, k_scale, v_scale, block_table, lengths, pa.I8)
        workspace = torch.empty(max(1, pa.attention_kv8_tree_workspace_bytes(x[:, :16], k, block_table, tokens)), dtype=torch.uint8, device="cuda")

        def step():
            pa.draft_tree(parents, 2, out=tree)
            pa.kvcache_append_rope(x[:, :16], x[:, 16:20], x[:, 20:], *cache, turns, tree=tree, out=x[:, :16])
            pa.attention_kv8_tree(x[:, :16], *cache, tree, out=out, workspace=workspace)
            pa.kvcache_keep(kept, *cache, max_tokens=tokens, out=after)
        step()
        torch.cuda.synchronize()
        before, free = torch.cuda.memory_stats()["allocation.all.allocated"], torch.cuda.mem_get_info()[0]
        step()
        torch.cuda.synchronize()
        assert torch.cuda.memory_stats()["allocation.all.allocated"] == before and torch.cuda.mem_get_info()[0] == free


def test_a_captured_step_serves_any_lengths_and_trees(pa):  # noqa: F811
    """The four calls in one graph, replayed with other lengths, parents and paths, against the same calls one by one."""
    g = torch.Generator(device="cuda").manual_seed(5)
    layers = [al.AttentionLayer(pa, width=256, heads=8, kv_heads=2, head_dim=64, sequences=2, longest=300, page_size=16, code_type=pa.I8) for _ in range(2)]
    x = torch.randn((24, 256), generator=g, device="cuda").bfloat16()
    parents = torch.full((24,), -1, dtype=torch.int32, device="cuda")
    kept = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([12, 12], dtype=torch.int32, device="cuda")

    def step(layer):
        tree = pa.draft_tree(parents, 2)
        y = layer.drafted(x, tree, lengths)
        return y, layer.keep(kept, lengths, 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(layers[0])
    for layer in layers:
        for t in (layer.k, layer.v, layer.k_scale, layer.v_scale):
            t.zero_()
    for i in range(5):
        x.copy_(torch.randn((24, 256), generator=g, device="cuda"))
        parents.copy_(torch.cat([torch.tensor([int(torch.randint(-1, max(n, 1), (1,))) if n else -1 for n in range(12)]) for _ in range(2)]))
        kept.copy_(torch.tensor([[0, 3 + i, 11, -1], [i, -1, -1, -1]]))
        graph.replay()
        y, after = step(layers[1])
        assert torch.equal(captured[0], y) and torch.equal(captured[1], after), i
        for n in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(layers[0], n).view(torch.uint8), getattr(layers[1], n).view(torch.uint8)), (i, n)
        lengths.copy_(after + 12)


def _calls(p):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((6, 12, 64), generator=g, device="cuda").bfloat16()
    positions = torch.tensor([0, 3, 9, 1, 31, 30], dtype=torch.int32, device="cuda")
    turns, narrow = p.rope_table(80, 64), p.rope_table(80, 24)
    k, v = (torch.randint(-100, 101, (8, 2, 16, 64), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.rand((8, 2), generator=g, device="cuda") * 0.01 for _ in range(2))
    table = torch.randperm(8, generator=g, device="cuda").to(torch.int32).view(2, 4)
    lengths = torch.tensor([60, 17], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    cache = (k, v, ks, vs, table, lengths, p.I8)
    parents = torch.tensor([-1, 0, -1, 0, 0, 1], dtype=torch.int32, device="cuda")
    tree = torch.tensor([[1], [3], [1], [3], [5], [11]], dtype=torch.int64, device="cuda")
    q, kn, vn = x[:, :8], x[:, 8:10], x[:, 10:]
    ragged = {"cu_tokens": cu, "max_tokens": 4}
    kept = torch.tensor([[0, 1, -1], [0, 2, 3]], dtype=torch.int32, device="cuda")
    return {
        "draft_tree": [((parents, 2), {}), ((parents, 2), ragged), ((parents, 2), {"out": torch.zeros((6, 3), dtype=torch.int64, device="cuda")}), ((parents.long(), 2), {}),
                       ((parents, 4), {}), ((parents, 2), {"cu_tokens": cu}), ((parents, 2), {"out": torch.zeros((5, 1), dtype=torch.int64, device="cuda")}),
                       ((parents.cpu(), 2), {}), ((parents, 0), {}), ((parents, 2, cu, 2), {}), ((parents, 2, None, 3, torch.cuda.current_stream()), {})],
        "kvcache_append_rope": [((q, kn, vn, *cache, turns), {}), ((q, kn, vn, *cache, turns), {**ragged, "tree": tree}), ((q, kn, vn, *cache, turns, positions), {}),
                                ((q, kn, vn, *cache, narrow), {"interleaved": True}), ((q.float(), kn.float(), vn.float(), *cache, turns), {}),
                                ((None, kn, vn, *cache, turns), {}), ((q, kn, vn, *cache, turns, positions, tree), {}), ((q.half(), kn, vn, *cache, turns), {}),
                                ((q, kn, vn, *cache, turns), {"tree": tree.int()}), ((q, kn, vn, *cache, turns), {"tree": tree[:5]}),
                                ((q, kn, vn, *cache, turns), {"positions": positions.long()}), ((q, kn, vn, *cache, turns[:, ::2]), {}), ((q[:5], kn, vn, *cache, turns), {}),
                                ((q, kn, vn, *cache, turns), {"out": torch.zeros((6, 8, 64), dtype=torch.bfloat16, device="cuda")}), ((q, kn, vn, *cache[:-1], 99, turns), {})],
        "attention_kv8_tree": [((q, *cache, tree), {}), ((q, *cache, tree), {**ragged, "want_lse": True}), ((q.half(), *cache, tree), {"window": 5, "scale": 0.1}),
                               ((q, *cache, tree), {"max_length": 60}), ((q, *cache, tree), {"out": torch.zeros((6, 8, 64), dtype=torch.bfloat16, device="cuda")}),
                               ((q.float(), *cache, tree), {}), ((q, *cache, None), {}), ((q, *cache, tree[:, 0]), {}), ((q, *cache, tree), {"window": 2}),
                               ((q[:, :7], *cache, tree), {}), ((q, *cache, tree), {"cu_tokens": cu}), ((q, *cache, tree), {"scale": -1.0}),
                               ((q, *cache, tree), {"workspace": torch.empty(64, dtype=torch.uint8, device="cuda"), "want_lse": True})],
        "kvcache_keep": [((kept, *cache), {"max_tokens": 3}), ((kept, *cache), ragged), ((kept, *cache), {}), ((kept.long(), *cache), {"max_tokens": 3}),
                         ((kept, *cache), {"max_tokens": 300}), ((kept, *cache), {"max_tokens": 3, "out": lengths}), ((kept[:1], *cache), {"max_tokens": 3}),
                         ((kept, *cache), {"max_tokens": 3, "out": torch.zeros(2, dtype=torch.int32, device="cuda")}), ((kept[:, :2], *cache), {"max_tokens": 3})],
    }


@pytest.mark.parametrize("name", ["draft_tree", "kvcache_append_rope", "attention_kv8_tree", "kvcache_keep"])
def test_native_calls_give_what_the_functions_give(pa, name):  # noqa: F811
    f = getattr(pa, name)
    assert f is not f.__wrapped__
    for i in range(len(_calls(pa)[name])):
        got, caches = [], []
        for g in (f, f.__wrapped__):
            args, kw = _calls(pa)[name][i]  # (of their own: a call changes its operands)
            try:
                r = g(*args, **kw)
            except Exception as e:  # noqa: BLE001
                r = (type(e), str(e))
            got.append(r)
            caches.append([t for t in args if isinstance(t, torch.Tensor)])
        flat = [list(r) if isinstance(r, tuple) else [r] for r in got]
        for a, b in zip(*flat):
            if isinstance(a, torch.Tensor):
                assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), (name, i)
            else:
                assert a == b, (name, i, a, b)
        assert all(torch.equal(a, b) for a, b in zip(*caches)), (name, i)
