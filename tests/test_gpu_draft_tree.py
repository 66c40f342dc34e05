"""Rows of bits from parents against sets."""
import pytest
import torch

import drafted_reference as dr
import kv8_reference as ref
from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[1], [2, 0, 1], [64] * 3, [65, 3], [24] * 16, [128, 100, 0, 7], [129], [256, 1, 255, 200], [63] * 70])
@pytest.mark.parametrize("width", [0, 1, 3])
def test_rows_are_ancestors(pa, counts, width):  # noqa: F811
    """Any parents, chains (width 1: each token behind the one before, or begun anew) and deep trees."""
    parents = dr.parents_of(counts, len(counts), width)
    if width == 1:
        parents[0] = list(range(-1, counts[0] - 1))  # (the longest path)
    words = -(-max(counts) // 64)
    rows = pa.draft_tree(dr.flat(parents), len(counts), cu_tokens=ref.starts(counts), max_tokens=max(counts))
    assert rows.shape == (sum(counts), words) and rows.dtype == torch.int64
    assert torch.equal(rows, dr.rows_of(dr.ways_of(parents), words))
    if len(set(counts)) == 1:
        assert torch.equal(pa.draft_tree(dr.flat(parents), len(counts)), rows)


def test_parents_that_are_none(pa):  # noqa: F811
    parents = [[-1, 0, 5, 2, -2, 4, 6, 2 ** 31 - 1, -2 ** 31, 1, 8], [0, 0], [1, -1]]
    counts = [len(p) for p in parents]
    rows = pa.draft_tree(dr.flat(parents), 3, cu_tokens=ref.starts(counts), max_tokens=11)
    ways = dr.ways_of(parents)
    assert ways[0][2] == set() and ways[0][3] == {3} and ways[0][5] == {5}
    assert torch.equal(rows, dr.rows_of(ways, 1))


def test_padded_batches_and_wider_rows(pa):  # noqa: F811
    """Rows that no sequence has, before the first, behind the last and beyond max_tokens, are left alone; words that no token needs are 0."""
    counts = [5, 0, 70]
    parents = dr.parents_of(counts, 3)
    wide = torch.full((90,), 3, dtype=torch.int32, device="cuda")
    wide[4:79] = dr.flat(parents)
    out = torch.full((90, 4), 77, dtype=torch.int64, device="cuda")
    pa.draft_tree(wide, 3, cu_tokens=ref.starts(counts) + 4, max_tokens=200, out=out)
    assert torch.equal(out[4:79], dr.rows_of(dr.ways_of(parents), 4)) and bool((out[:4] == 77).all()) and bool((out[79:] == 77).all())
    out.fill_(77)
    pa.draft_tree(wide, 3, cu_tokens=ref.starts(counts) + 4, max_tokens=66, out=out)
    assert torch.equal(out[4:75], dr.rows_of(dr.ways_of([parents[0], [], parents[2][:66]]), 4)) and bool((out[75:] == 77).all())
    # starts that are no starts: nothing outside the operands is touched
    for cu in ([0, 200, 90, 95], [-5, -1, 50, 20], [90, 90, 90, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        pa.draft_tree(wide, 3, cu_tokens=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_tokens=70, out=out)
    torch.cuda.synchronize()


def test_captured_and_on_another_stream(pa):  # noqa: F811
    counts = [100] * 5
    parents = [dr.flat(dr.parents_of(counts, seed)) for seed in range(4)]
    want = [dr.rows_of(dr.ways_of(dr.parents_of(counts, seed)), 2) for seed in range(4)]
    now = parents[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = pa.draft_tree(now, 5)
    for p, w in zip(parents, want):
        now.copy_(p)
        graph.replay()
        assert torch.equal(rows, w)
    side = torch.cuda.Stream()
    out = torch.empty_like(rows)
    torch.cuda.synchronize()
    pa.draft_tree(parents[1], 5, stream=side, out=out)
    side.synchronize()
    assert torch.equal(out, want[1])
