"""Which keys a query of the attention over an 8-bit cache sees: the arithmetic that its kernels run, compiled for the host."""
import ctypes
import os

import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "pto_kernels", "build", "libkv8places.so")
MOST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def places():
    assert os.path.exists(LIB), "build the test libraries first: make -C tests/pto_kernels"
    return ctypes.CDLL(LIB)


@pytest.mark.parametrize("causal", [False, True])
def test_keys_by_their_definition(places, causal):
    """0 <= j < length, j <= place (causal), j > place - window (window > 0): lengths, new tokens and windows from none to as many as 32 bits hold,
    queries before the first key among them."""
    x, y = ctypes.c_int(), ctypes.c_int()
    for length in (0, 1, 2, 5, 16, 31, 1000, 2 ** 31 - 2 ** 20):
        for count in (1, 2, 3, 9, 16, 4097, 2 ** 30, MOST):
            for nth in {0, 1, count // 2, count - 1}:
                place = length - count + nth
                for window in (0, 1, 2, 5, 17, 1000, 2 ** 30, 2 ** 31 - 2 ** 20, MOST - 1, MOST):
                    first = max(place - window + 1, 0) if window else 0
                    end = min(length, max(place + 1, 0)) if causal else length
                    assert places.kv8_first_key(place, window) == first, (length, count, nth, window)
                    places.kv8_keys_of(place, length, int(causal), window, ctypes.byref(x), ctypes.byref(y))
                    assert (x.value, y.value) == (first, max(end, first)), (length, count, nth, window)
                    assert 0 <= x.value <= max(length, place + 1) and x.value <= y.value <= max(length, x.value)


@pytest.mark.parametrize("shift", [4, 5, 6, 7, 8])
def test_the_most_pages_of_so_many_tokens(places, shift):
    page = 1 << shift
    for tokens in (1, 2, page - 1, page, page + 1, page + 2, 10 * page, 10 * page + 1, 2 ** 30 + 3, MOST - page, MOST - 1, MOST):
        most = max((start + tokens - 1) // page - start // page + 1 for start in (0, 1, 2, page // 2, page - 2, page - 1))
        assert places.kv8_pages_of(tokens, shift) == most, tokens


def test_more_tokens_a_sequence_than_there_are():
    """max_tokens bounds the sequences' tokens and may be loose; no sequence has more than all tokens, which is what work is planned for."""
    import __graft_entry__ as ge
    pa = ge.load_package()
    lib = pa.lib()
    for heads, kv_heads, dim, tokens in ((8, 8, 128, 4), (64, 8, 128, 4), (64, 8, 64, 300), (16, 2, 256, 70)):
        cache = pa._Kv8Cache(pages=4096, kv_heads=kv_heads, page_size=64, head_dim=dim, sequences=2, max_pages=512)
        need = [lib.ptoamd_attention_kv8_workspace_bytes(ctypes.byref(cache), heads, tokens, most, 0, window) for window in (0, 1000) for most in (tokens, tokens + 1, 2 ** 20, MOST)]
        assert need[0] > 0 and set(need[:4]) == {need[0]} and set(need[4:]) == {need[4]}, need


def test_tables_of_nearly_as_many_places_as_32_bits_hold():
    """Kernels step past a sequence's last key by up to 1040 places; a table whose places leave no room for that is refused."""
    from test_kv8_refusals import call
    for name in ("ptoamd_kvcache_append", "ptoamd_attention_kv8"):
        for page, pages in ((256, 2 ** 23 - 1), (256, 2 ** 23 - 4), (16, 2 ** 27 - 16), (64, 2 ** 25 - 1023)):
            rc, error = call(name, cache_page_size=page, cache_max_pages=pages, tokens=0, most=0)
            assert rc == -2 and "too many" in error, (name, page, pages, rc)
        for page, pages in ((256, 2 ** 23 - 256), (16, 2 ** 27 - 4096)):
            assert call(name, cache_page_size=page, cache_max_pages=pages, tokens=0, most=0)[0] == 0


def test_more_rows_than_32_bits_number():
    """A sequence's new tokens times the query heads of a key head are rows, numbered in 32 bits."""
    from test_kv8_refusals import AT, call
    for heads, tokens in ((65534, 2 ** 17), (64, 2 ** 28)):
        for cu in (None, AT):
            rc, error = call("ptoamd_attention_kv8", heads=heads, tokens=tokens if cu else 2 * tokens, most=tokens, cu=cu)
            assert rc == -2 and "rows" in error, (rc, error)
