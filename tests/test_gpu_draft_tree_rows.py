"""The rows that a call of draft_tree gives to tokens of no sequence: empty ones in a result of its own, whatever its memory held."""
import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


def dirty(*shape):
    """The allocator's next block of that size holds ones."""
    torch.full(shape, -1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()


@pytest.mark.parametrize("form", ["native", "function"])
@pytest.mark.parametrize("most", [0, 1, 40, 66, 70, 200])
@pytest.mark.parametrize("counts,before,behind", [([5, 0, 70], 4, 11), ([0, 0, 0], 3, 70), ([70], 0, 0), ([1] * 40 + [70], 0, 1000), ([0, 70, 0], 500, 0)])
def test_rows_of_no_sequence_are_empty(pa, form, most, counts, before, behind):  # noqa: F811
    draft = pa.draft_tree if form == "native" else pa.draft_tree.__wrapped__
    parents = dr.parents_of(counts, 3)
    tokens = before + sum(counts) + behind
    wide = torch.full((tokens,), 3, dtype=torch.int32, device="cuda")
    wide[before:before + sum(counts)] = dr.flat(parents)
    words = max(1, -(-min(most, tokens) // 64))
    want = torch.zeros((tokens, words), dtype=torch.int64, device="cuda")
    at = before
    for mine in parents:
        if mine[:most]:
            want[at:at + len(mine[:most])] = dr.rows_of(dr.ways_of([mine[:most]]), words)
        at += len(mine)
    cu = ref.starts(counts) + before
    for _ in range(3):
        dirty(tokens, words)
        got = draft(wide, len(counts), cu_tokens=cu, max_tokens=most)
        assert got.shape == want.shape and torch.equal(got, want)
        del got


def test_starts_that_are_no_starts_touch_nothing_else(pa):  # noqa: F811
    parents = torch.full((90,), -1, dtype=torch.int32, device="cuda")
    for cu in ([0, 200, 90, 95], [-5, -1, 50, 20], [90, 90, 90, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [2 ** 31 - 1] * 4):
        whole = torch.full((94, 2), 77, dtype=torch.int64, device="cuda")
        rc = pa.lib().ptoamd_draft_tree_all(whole[2:].data_ptr(), 2, parents.data_ptr(), 90, 3, torch.tensor(cu, dtype=torch.int32, device="cuda").data_ptr(), 70,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert bool((whole[:2] == 77).all()) and bool((whole[92:] == 77).all())


def test_captured(pa):  # noqa: F811
    parents = torch.full((90,), -1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([3, 20, 60, 80], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = pa.draft_tree(parents, 3, cu_tokens=cu, max_tokens=64)
    for starts in ([0, 0, 64, 90], [9, 9, 9, 9], [1, 60, 88, 90], [0, 30, 60, 90]):
        cu.copy_(torch.tensor(starts))
        rows.fill_(-1)
        graph.replay()
        want = torch.zeros_like(rows)
        for lo, hi in zip(starts[:-1], starts[1:]):
            for i in range(lo, min(hi, lo + 64)):
                want[i, 0] = 1 << (i - lo) if i - lo < 63 else -2 ** 63
        assert torch.equal(rows, want), starts
