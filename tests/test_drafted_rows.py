"""Drafted tokens' rows of bits as the attention kernels hold them, cleared behind a sequence's last token, and what they read from them; compiled for the host."""
import random

import pytest

from test_drafted_bits import MOST, drafted, row  # noqa: F401


def cleared(drafted, mine, words, count, held):  # noqa: F811
    """The words that a kernel holds of a row, more than it has where rows are short."""
    return (type(mine)._type_ * held)(*[drafted.drafted_own_word(mine, words, w, count) & 0xFFFFFFFF for w in range(held)])


@pytest.mark.parametrize("words,held", [(2, 2), (2, 8), (6, 6), (8, 8)])
def test_bits_of_tokens_that_there_are(drafted, words, held):  # noqa: F811
    rng = random.Random(words + held)
    for bits in (0, 2 ** (32 * words) - 1, rng.getrandbits(32 * words)):
        for count in {0, 1, 31, 32, 33, 63, 64, 32 * words - 1, 32 * words}:
            got = cleared(drafted, row(bits, words), words, count, held)
            assert sum(w << (32 * i) for i, w in enumerate(got)) == bits & (2 ** count - 1), (bits, count)


@pytest.mark.parametrize("count", [1, 5, 32, 33, 64, 100, 256])
def test_keys_by_their_definition(drafted, count):  # noqa: F811
    """first <= j < old, or old <= j < length and bit j - old; tokens that have no place (old < 0) among them, bits behind the last token, tiles behind the last key."""
    rng = random.Random(count)
    words = 2 * (-(-count // 64))
    for length in (0, 1, count - 1, count, count + 1, count + 40, count + 1000, MOST):
        old = length - count
        for bits in (0, 2 ** (32 * words) - 1, rng.getrandbits(32 * words)):
            mine = row(bits, words)
            for held in {words, 8}:
                own = cleared(drafted, mine, words, count, held)
                for first in {0, max(old - 5, 0), max(old, 0), max(old - 300, 0), 2 ** 31 - 1}:
                    for key in {0, 16, max(old - 48, 0), max(old - 17, 0), max(old - 1, 0), max(old, 0), max(old + 30, 0), max(length - 20, 0), length, length // 2, length + 1040}:
                        want = 0
                        for b in range(32):
                            j = key + b
                            if first <= j < old or (old <= j < length and bits >> (j - old) & 1):
                                want |= 1 << b
                        assert drafted.drafted_seen_by_own(own, held, key, first, old) & 0xFFFFFFFF == want, (length, first, key)
                        if first <= max(old, 0):
                            assert drafted.drafted_seen_keys(mine, words, key, first, old, length) == want, (length, first, key)


@pytest.mark.parametrize("count", [1, 33, 64, 256])
def test_a_window_goes_by_the_others_that_are_seen(drafted, count):  # noqa: F811
    rng = random.Random(count)
    words = 2 * (-(-count // 64))
    for bits in (0, 2 ** (32 * words) - 1, rng.getrandbits(32 * words)):
        for self in {0, count // 2, count - 1}:
            others = sum(1 for t in range(count) if t != self and bits >> t & 1)
            for old in (-count, -1, 0, 1, 300, 5000, MOST - count):
                for window in (0, count, 300, 4097, 2 ** 31 - 1):
                    want = max(0, old + others + 1 - window) if window else 0
                    assert drafted.drafted_first_of_older(row(bits, words), words, count, self, old, window) == want, (self, old, window)
