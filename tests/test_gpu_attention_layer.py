"""The operators around an 8-bit cache together: rope, append and attention between two products, prompts in chunks and a captured step."""
import os
import sys

import pytest
import torch

from test_gpu_parity import pa  # noqa: F401

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import attention_layer as al  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,dim,error", [("E4M3", 128, 0.06), ("E4M3", 64, 0.06), ("I8", 128, 0.02), ("I8", 256, 0.02)])
def test_a_layer_serves_prompts_and_steps(pa, code, dim, error):  # noqa: F811
    """The relative error of a result is that of its inputs.  E4M3 codes: three bits behind the point, a step of 2^-3 of a value's power of two, so
    2^-3 / sqrt(12) = 0.036 of values beside one, 0.026 of the mean square over an octave; keys and values each.  int8: a page's largest over
    127 a step; of normal values whose largest is 4.2 deviations, 4.2 / 127 / sqrt(12) = 0.0096.  Keys reach the result through scores of some
    1 +- 0.026 (0.0096), weights that average values of random signs: both errors add in squares, 0.037 and 0.0136; bf16's three roundings
    (2^-9 / sqrt(3) = 0.0011 each) are nothing beside them.  Bounds: half as much again."""
    layer = al.AttentionLayer(pa, width=512, heads=8, kv_heads=2, head_dim=dim, sequences=3, longest=400, code_type=getattr(pa, code))
    g = torch.Generator(device="cuda").manual_seed(2)
    prompts = [torch.randn((n, 512), generator=g, device="cuda").bfloat16() for n in (390, 71, 7)]
    outs = al.serve(layer, prompts, chunk=96, steps=5)
    assert al.relative_error(layer, prompts, outs) < error


def test_a_step_allocates_nothing_beside_its_results(pa):  # noqa: F811
    """With out and a workspace given, the three calls allocate no device memory, in torch or behind its back."""
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.zeros((64, 4, 64, 128), dtype=torch.int8, device="cuda") for _ in range(2))
    k_scale, v_scale = (torch.zeros((64, 4), device="cuda") for _ in range(2))
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    lengths = torch.tensor([2048, 100], dtype=torch.int32, device="cuda")
    turns = pa.rope_table(2048, 128)
    for tokens in (1, 70):
        x = torch.randn((2 * tokens, 24, 128), generator=g, device="cuda").bfloat16()
        positions = torch.arange(2 * tokens, dtype=torch.int32, device="cuda")
        out = torch.empty((2 * tokens, 16, 128), dtype=torch.bfloat16, device="cuda")
        cache = (k, v, k_scale, v_scale, table, lengths, pa.I8)
        workspace = torch.empty(pa.attention_kv8_workspace_bytes(x[:, :16], k, table, tokens), dtype=torch.uint8, device="cuda")
        assert workspace.numel() > 0

        def step():
            pa.rope(x[:, :20], turns, positions, out=x[:, :20])
            pa.kvcache_append(x[:, 16:20], x[:, 20:], *cache)
            pa.attention_kv8(x[:, :16], *cache, out=out, workspace=workspace)
        step()
        torch.cuda.synchronize()
        before, free = torch.cuda.memory_stats()["allocation.all.allocated"], torch.cuda.mem_get_info()[0]
        step()
        torch.cuda.synchronize()
        assert torch.cuda.memory_stats()["allocation.all.allocated"] == before and torch.cuda.mem_get_info()[0] == free
        assert "split" in pa.last_kernel() or "join" in pa.last_kernel()


def _calls(p):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((6, 12, 64), generator=g, device="cuda").bfloat16()
    positions = torch.tensor([0, 3, 9, 1, 31, 40], dtype=torch.int32, device="cuda")
    turns, narrow = p.rope_table(32, 64), p.rope_table(32, 48)
    k, v = (torch.randint(-100, 101, (8, 2, 16, 64), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.rand((8, 2), generator=g, device="cuda") * 0.01 for _ in range(2))
    table = torch.randperm(8, generator=g, device="cuda").to(torch.int32).view(2, 4)
    lengths = torch.tensor([60, 17], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    cache = (k, v, ks, vs, table, lengths, p.I8)
    q = x[:, :8]
    return {
        "rope": [((x, turns, positions), {}), ((x, narrow, positions, True), {}), ((x, turns, positions), {"backward": True}), ((x[:, 2:5], turns, positions), {}),
                 ((x.float(), turns, positions), {"out": torch.zeros((6, 12, 64), device="cuda")}), ((x, turns, positions.long()), {}), ((x[0], turns, positions), {}),
                 ((x, turns[:, ::2], positions), {}), ((x, turns, positions, False, False, torch.cuda.current_stream()), {}), ((x, p.rope_table(32, 128), positions), {}),
                 ((x.cpu(), turns, positions), {})],
        "kvcache_append": [((x[:, 8:10], x[:, 10:], *cache), {}), ((x[:, 8:10], x[:, 10:], *cache), {"cu_tokens": cu, "max_tokens": 4}),
                           ((x[:, 8:10].float(), x[:, 10:].float(), *cache), {}), ((x[:, 8:10], x[:, 10:].half(), *cache), {}),
                           ((x[:5, 8:10], x[:5, 10:], *cache), {}), ((x[:, 8:10], x[:, 10:], *cache[:-1], 99), {}), ((x[:, 8:9], x[:, 10:], *cache), {})],
        "attention_kv8": [((q, *cache), {}), ((q, *cache), {"cu_tokens": cu, "max_tokens": 4, "want_lse": True}), ((q.half(), *cache), {"window": 5, "scale": 0.1}),
                          ((q, *cache), {"causal": False, "max_length": 60}), ((q, *cache), {"out": torch.zeros((6, 8, 64), dtype=torch.bfloat16, device="cuda")}),
                          ((q.float(), *cache), {}), ((q[:, :7], *cache), {}), ((q, *cache), {"cu_tokens": cu}), ((q, *cache), {"scale": -1.0}),
                          ((q[:, :, :56], *cache), {}), ((q, *cache), {"workspace": torch.empty(64, dtype=torch.uint8, device="cuda"), "want_lse": True})],
    }


@pytest.mark.parametrize("name", ["rope", "kvcache_append", "attention_kv8"])
def test_native_calls_give_what_the_functions_give(pa, name):  # noqa: F811
    f = getattr(pa, name)
    assert f is not f.__wrapped__
    for i in range(len(_calls(pa)[name])):
        got, caches = [], []
        for g in (f, f.__wrapped__):
            args, kw = _calls(pa)[name][i]  # (of their own: an append changes its operands)
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
