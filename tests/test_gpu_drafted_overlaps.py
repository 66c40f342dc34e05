"""Results of the append with rotation beside its operands in one tensor, where they share no element: as with a tensor of their own."""
import pytest
import torch

import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def fresh():
    return ref.Cache("i8", [40, 33], 4, 64, 16, 3)


@pytest.mark.parametrize("layout", ["fused", "interleaved", "spare heads", "interleaved spare"])
def test_in_one_tensor(pa, layout):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((10, 24, 64), generator=g, device="cuda").bfloat16()
    parts = {"fused": (slice(0, 8), slice(8, 12), slice(12, 16), slice(0, 8)), "interleaved": (slice(0, 12, 3), slice(1, 12, 3), slice(2, 12, 3), slice(0, 12, 3)),
             "spare heads": (slice(0, 8), slice(8, 12), slice(12, 16), slice(16, 24)),
             "interleaved spare": (slice(0, 16, 4), slice(1, 16, 4), slice(2, 16, 4), slice(3, 16, 4))}[layout]
    q, k, v, out = (x[:, p] for p in parts)
    table = pa.rope_table(64, 64)
    apart, together = fresh(), fresh()
    want = pa.kvcache_append_rope(q.clone(), k.clone(), v.clone(), *apart.operands(pa), table)
    before = x.clone()
    got = pa.kvcache_append_rope(q, k, v, *together.operands(pa), table, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(apart, n).view(torch.uint8), getattr(together, n).view(torch.uint8)), n
    out.copy_(before[:, parts[3]])
    assert torch.equal(x, before)


def test_over_other_rows_is_refused(pa):  # noqa: F811
    x = torch.randn((11, 16, 64), device="cuda").bfloat16()
    cache, table = fresh(), pa.rope_table(64, 64)
    for out in (x[1:, :8], x[:10, 1:9], x[:10, 4:12]):
        with pytest.raises(pa.PtoAmdError, match="overlap"):
            pa.kvcache_append_rope(x[:10, :8], x[:10, 8:12], x[:10, 12:], *cache.operands(pa), table, out=out)
