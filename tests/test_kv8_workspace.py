"""The workspace of attention over an 8-bit cache stays bounded whatever the host's bounds are (no GPU: sizes alone choose it)."""
import ctypes
import random

import pytest

import __graft_entry__ as ge


def need(heads, kv_heads, dim, sequences, tokens, most, max_pages, max_length=0, window=0, page=64):
    pa = ge.load_package()
    cache = pa._Kv8Cache(pages=1, kv_heads=kv_heads, page_size=page, head_dim=dim, sequences=sequences, max_pages=max_pages)
    return pa._lib.ptoamd_attention_kv8_workspace_bytes(ctypes.byref(cache), heads, tokens, most, max_length, window)


@pytest.mark.parametrize("sequences,heads,kv_heads,dim,max_pages", [(256, 128, 8, 128, 2048), (382, 256, 32, 256, 663882), (65535, 8, 8, 64, 4096), (1, 8, 1, 64, 2 ** 24),
                                                                    (1, 1, 1, 16, 2 ** 25 - 1024)])
def test_few_rows_under_a_wide_table(sequences, heads, kv_heads, dim, max_pages):
    """A captured decode step plans for its table's width, whatever lengths it meets."""
    for tokens in (1, 3):
        assert need(heads, kv_heads, dim, sequences, sequences * tokens, tokens, max_pages) <= 256 << 20


def test_any_sizes():
    rng = random.Random(3)
    for _ in range(20000):
        kv, most, seqs = rng.choice([1, 2, 4, 8, 16, 32]), int(2 ** rng.uniform(0, 17)), int(2 ** rng.uniform(0, 9))
        tokens = seqs * most if rng.random() < 0.5 else max(most, int(seqs * most * rng.random()))
        args = (kv * rng.choice([1, 2, 4, 7, 8, 16, 64]), kv, rng.choice([64, 128, 256]), seqs, tokens, most, int(2 ** rng.uniform(0, 20)),
                rng.choice([0, 0, int(2 ** rng.uniform(5, 20))]), rng.choice([0, 0, rng.randrange(1, 100000)]))
        assert need(*args) <= 288 << 20, args  # (many rows: the parts that the mean tile of rows needs, some 271 MB at most)
