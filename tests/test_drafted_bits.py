"""Which keys a drafted token sees: the arithmetic that the kernels run on its row of bits, compiled for the host."""
import ctypes
import os
import random

import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "pto_kernels", "build", "libdrafted.so")
MOST = 2 ** 31 - 2 ** 16


@pytest.fixture(scope="module")
def drafted():
    assert os.path.exists(LIB), "build the test libraries first: make -C tests/pto_kernels"
    lib = ctypes.CDLL(LIB)
    lib.drafted_bits_below.restype = lib.drafted_row_bits.restype = lib.drafted_seen_keys.restype = ctypes.c_uint32
    return lib


def row(bits, words):
    return (ctypes.c_uint32 * words)(*[bits >> (32 * w) & 0xFFFFFFFF for w in range(words)])


def test_bits_below(drafted):
    for n in (-2 ** 31, -33, -32, -1, 0, 1, 5, 31, 32, 33, 2 ** 31 - 1):
        assert drafted.drafted_bits_below(n) == 2 ** min(max(n, 0), 32) - 1, n


@pytest.mark.parametrize("words", [2, 4, 6, 8])
def test_rows_from_any_bit(drafted, words):
    rng = random.Random(words)
    bits = rng.getrandbits(32 * words)
    mine = row(bits, words)
    for at in list(range(-70, 32 * words + 70)) + [-MOST, MOST, -2 ** 31, 2 ** 31 - 1]:
        want = sum(1 << b for b in range(32) if 0 <= at + b < 32 * words and bits >> (at + b) & 1)
        assert drafted.drafted_row_bits(mine, words, at) == want, at


@pytest.mark.parametrize("words", [2, 8])
def test_others_seen(drafted, words):
    rng = random.Random(words)
    for bits in (0, 2 ** (32 * words) - 1, rng.getrandbits(32 * words), rng.getrandbits(32 * words)):
        for count in {0, 1, 31, 32, 33, 32 * words - 1, 32 * words}:
            for self in {0, 1, 31, 32, 63, 32 * words - 1}:
                want = sum(1 for t in range(count) if t != self and bits >> t & 1)
                assert drafted.drafted_others_seen(row(bits, words), words, count, self) == want, (count, self)


@pytest.mark.parametrize("count", [1, 5, 32, 64, 100, 256])
def test_keys_by_their_definition(drafted, count):
    """first <= j < old, or old <= j < length and bit j - old; tokens that have no place (old < 0) among them, and bits behind the last token."""
    rng = random.Random(count)
    words = 2 * (-(-count // 64))
    for length in (0, 1, count - 1, count, count + 1, count + 40, count + 1000, MOST):
        old = length - count
        for bits in (0, 2 ** (32 * words) - 1, rng.getrandbits(32 * words)):
            for first in {0, max(old - 5, 0), max(old, 0), max(old - 300, 0)}:
                mine = row(bits, words)
                for key in {0, 16, max(old - 48, 0), max(old - 17, 0), max(old - 1, 0), max(old, 0), max(old + 30, 0), max(length - 20, 0), max(length, 0), length // 2}:
                    want = 0
                    for b in range(32):
                        j = key + b
                        if first <= j < old or (j >= old and j < length and j - old < 32 * words and bits >> (j - old) & 1):
                            want |= 1 << b
                    assert drafted.drafted_seen_keys(mine, words, key, first, old, length) == want, (length, first, key)
