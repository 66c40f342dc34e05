"""Whether two operands overlap, by their addresses and strides, against all their bytes."""
import ctypes
import os
import random

import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "pto_kernels", "build", "liboverlap.so")
AT = 1 << 40


@pytest.fixture(scope="module")
def meet():
    assert os.path.exists(LIB), "build the test libraries first: make -C tests/pto_kernels"
    lib = ctypes.CDLL(LIB)

    def f(a, x, b, y):
        got = [lib.overlap_meet(*(ctypes.c_uint64(p) if i % 2 == 0 else (ctypes.c_int64 * 5)(*p) for i, p in enumerate(pair))) for pair in ((a, x, b, y), (b, y, a, x))]
        assert got[0] == got[1], (a, x, b, y)
        return bool(got[0])
    return f


def covered(at, rows):
    tokens, heads, token, head, width = rows
    return {at + t * token + h * head + i for t in range(tokens) for h in range(heads) for i in range(width)}


def test_views_of_one_tensor(meet):
    """The same distances of tokens and heads: exact."""
    rng = random.Random(1)
    for _ in range(4000):
        width = rng.choice([1, 2, 4, 6])
        head = rng.choice([width, width, width + rng.randrange(5), 3 * width])
        token = head * rng.randrange(1, 9) + rng.randrange(3)
        x, y = ((rng.randrange(0, 6), rng.randrange(0, 5), token, head, width) for _ in range(2))
        b = AT + rng.randrange(-3 * token, 3 * token)
        assert meet(AT, x, b, y) == bool(covered(AT, x) & covered(b, y)), (x, b - AT, y)


def test_rows_and_a_piece_of_memory(meet):
    rng = random.Random(2)
    for _ in range(4000):
        width = rng.choice([1, 2, 4, 6])
        head = rng.choice([width, width + rng.randrange(5), 2 * width])
        x = (rng.randrange(0, 7), rng.randrange(0, 5), head * rng.randrange(1, 9) + rng.randrange(3), head, width)
        y = (1, 1, 0, 0, rng.randrange(0, 40))
        b = AT + rng.randrange(-60, 6 * x[2] + 60)
        assert meet(AT, x, b, y) == bool(covered(AT, x) & covered(b, y)), (x, b - AT, y)


def test_whole_tensors_of_other_shapes(meet):
    """Heads and tokens that lie together are one piece, whatever they are made of."""
    rng = random.Random(3)
    for _ in range(2000):
        rows = []
        for _ in range(2):
            width, heads = rng.choice([2, 4, 6]), rng.randrange(1, 5)
            rows.append((rng.randrange(1, 6), heads, heads * width, width, width))
        b = AT + rng.randrange(-150, 150)
        assert meet(AT, rows[0], b, rows[1]) == bool(covered(AT, rows[0]) & covered(b, rows[1])), (rows, b - AT)


def test_never_where_nothing_is_shared(meet):
    """Any strides, broadcast and descending ones among them."""
    rng = random.Random(4)
    for _ in range(6000):
        x, y = ((rng.randrange(1, 5), rng.randrange(1, 5), rng.randrange(-40, 40), rng.randrange(-12, 12), rng.randrange(1, 6)) for _ in range(2))
        b = AT + rng.randrange(-100, 100)
        if not covered(AT, x) & covered(b, y):
            assert not meet(AT, x, b, y), (x, b - AT, y)


def test_large_tensors(meet):
    head, token = 256, 96 * 256
    q, k = (1 << 20, 64, token, head, 256), (1 << 20, 8, token, head, 256)
    assert not meet(AT, q, AT + 64 * 256, k) and not meet(AT, q, AT + 72 * 256, k)
    assert meet(AT, q, AT + 63 * 256, k) and meet(AT, q, AT + 89 * 256, k) and not meet(AT, q, AT + 88 * 256, k)
    assert not meet(AT, q, AT + (1 << 20) * token, q) and meet(AT, q, AT + ((1 << 20) - 1) * token, q)
