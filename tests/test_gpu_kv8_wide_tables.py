"""Attention over an 8-bit cache under tables that are far wider than the sequences, and sequences as long as places go."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_attention_kv8 import queries
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("lengths", [[20011] + [1 + 7 * i % 61 for i in range(199)], [8192, 0, 5]])
def test_a_step_that_is_planned_for_the_table(pa, code, lengths):  # noqa: F811
    """Without max_length the table's 131072 places are what the work is cut by: fewer parts than a part for 4096 of them where the workspace's
    bound says so, and most of them empty."""
    heads = 64 if len(lengths) > 10 else 16
    cache = ref.Cache(code, lengths, 4, 128, 64, 51)
    wide = torch.full((len(lengths), 2048), -1, dtype=torch.int32, device="cuda")
    wide[:, :cache.table.shape[1]] = cache.table
    q = queries(len(lengths), heads, 128, torch.bfloat16, 52)
    expected = ref.attention(q, cache, [1] * len(lengths))
    cache.table = wide
    assert 0 < pa.attention_kv8_workspace_bytes(q, cache.k, wide, 1) <= 256 << 20
    out, lse = pa.attention_kv8(q, *cache.operands(pa), want_lse=True)
    assert pa.last_kernel() == "attention_kv8_few_split"
    ref.check_attention(out, expected, lse)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("short", [0, 1, 255, 1000])
def test_the_longest_sequence(pa, code, short):  # noqa: F811
    """2^31 - 2^16 places, less a few, of one page that the whole table names: the result is the page's own, every key as often as it comes, the
    log-sum larger by the logarithm of that.  Sums of f32 in a row: 128 turns of a wave, 4096 parts of a group of lanes, and their join, 2^-24 each."""
    page, dim, pages = 256, 16, 2 ** 23 - 256
    one = ref.Cache(code, [page], 1, dim, page, 53)
    q = queries(1, 2, dim, torch.bfloat16, 54)
    table = torch.full((1, pages), int(one.table[0, 0]), dtype=torch.int32, device="cuda")
    length = page * pages - short
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    print("longest", code, short, flush=True)
    out, lse = pa.attention_kv8(q, one.k, one.v, one.k_scale, one.v_scale, table, lengths, one.operands(pa)[-1], want_lse=True)
    expected, norm, mag, spread = ref.attention(q, one, [1], causal=False)
    sums = (128 + 4096 + 32) * 2.0 ** -24
    # (`short` of 2^31 keys are missing: a share of 2^-21 of the weights at most)
    norm = norm + math.log(pages)
    tol = 2.0 ** -8 * expected.abs() + (2.0 ** -11 + 2 * sums + 2.0 ** -19 * spread[:, :, None]) * mag
    assert bool(((out.double() - expected).abs() <= tol).all())
    assert bool(((lse.double() - norm).abs() <= sums + 2.0 ** -20 * (spread + norm.abs()) + 2.0 ** -19).all()), float((lse.double() - norm).abs().max())
