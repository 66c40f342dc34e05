"""attention_kv8 on streams that are not the current one."""
import pytest
import torch

import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 70])
def test_calls_on_two_streams_have_workspaces_of_their_own(pa, tokens):  # noqa: F811
    """Split calls on two streams and allocations on a third, nothing waited for in between: as the same calls one by one, bit for bit.  (Results are
    given: a block that a fill on the current stream still writes must not become one of another stream's.)"""
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for seed in (21, 22):
        cache = ref.Cache("e4m3", [9000, 500], 2, 128, 64, seed)
        q = torch.randn((2 * tokens, 16, 128), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
        need = pa.attention_kv8_workspace_bytes(q, cache.k, cache.table, tokens)
        assert need > 0
        work.append((cache, q, pa.attention_kv8(q, *cache.operands(pa), want_lse=True), need))
        ref.check_attention(work[-1][2][0], ref.attention(q, cache, [tokens] * 2), work[-1][2][1])
    got = [[torch.empty_like(q) for _ in range(20)] for _, q, _, _ in work]
    torch.cuda.synchronize()
    for i in range(20):
        for (cache, q, _, need), side, outs in zip(work, sides, got):
            pa.attention_kv8(q, *cache.operands(pa), out=outs[i], stream=side)
            torch.empty(need, dtype=torch.uint8, device="cuda").fill_(0xFF)  # (the current stream's next owner of such a block)
    torch.cuda.synchronize()
    for (_, _, expected, _), outs in zip(work, got):
        for i, out in enumerate(outs):
            assert torch.equal(out, expected[0]), i


def test_a_stream_by_its_handle(pa):  # noqa: F811
    import types
    cache = ref.Cache("i8", [9000], 2, 128, 64, 23)
    q = torch.randn((1, 16, 128), generator=torch.Generator(device="cuda").manual_seed(24), device="cuda").bfloat16()
    expected = pa.attention_kv8(q, *cache.operands(pa))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = pa.attention_kv8(q, *cache.operands(pa), stream=types.SimpleNamespace(cuda_stream=side.cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, expected)
