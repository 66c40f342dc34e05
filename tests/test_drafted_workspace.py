"""The workspace of attention of drafted tokens stays bounded whatever the host's bounds are (no GPU: sizes alone choose it)."""
import ctypes
import random

import __graft_entry__ as ge


def test_any_sizes():
    pa, rng = ge.load_package(), random.Random(3)
    for _ in range(20000):
        kv, most, seqs = rng.choice([1, 2, 4, 8, 16, 32, 160]), int(2 ** rng.uniform(0, 8.01)), int(2 ** rng.uniform(0, 16))
        tokens = seqs * most if rng.random() < 0.5 else max(most, int(seqs * most * rng.random()))
        page = rng.choice([16, 64, 256])
        cache = pa._Kv8Cache(pages=1, kv_heads=kv, page_size=page, head_dim=rng.choice([16, 64, 80, 128, 256]), sequences=seqs,
                             max_pages=int(2 ** rng.uniform(0, 30)) // page + 1)
        args = (kv * rng.choice([1, 2, 4, 7, 8, 16, 64]), tokens, most, rng.choice([0, 0, int(2 ** rng.uniform(5, 30))]), rng.choice([0, 0, rng.randrange(256, 100000)]))
        need = pa._lib.ptoamd_attention_kv8_tree_workspace_bytes(ctypes.byref(cache), *args)
        assert need <= 288 << 20, (seqs, kv, cache.head_dim, page, cache.max_pages, args)
