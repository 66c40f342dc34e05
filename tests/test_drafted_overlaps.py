"""Results of the calls around drafted trees over operands that other workgroups still read are refused, before anything is launched."""
import ctypes

import pytest

import __graft_entry__ as ge
from test_kv8_refusals import AT

FAR = 1 << 20  # between operands
OPERANDS = ["q", "k", "v", "table", "positions", "tree", "cu", "lengths", "block_table", "k_scale", "v_scale", "kc", "vc", "out"]


def places(**change):
    """Addresses far from each other, but those given."""
    at = {name: AT + i * FAR for i, name in enumerate(OPERANDS)}
    at.update(change)
    return at


def cache_at(pa, at):
    return pa._Kv8Cache(k=at["kc"], v=at["vc"], k_scale=at["k_scale"], v_scale=at["v_scale"], block_table=at["block_table"], lengths=at["lengths"], code_type=pa.I8, pages=4,
                        kv_heads=2, page_size=16, head_dim=64, sequences=2, max_pages=2, k_page_stride=2048, k_head_stride=1024, k_token_stride=64, v_page_stride=2048,
                        v_head_stride=1024, v_token_stride=64)


def append(at, which, q=(256, 64), out=(256, 64), k=(128, 64), v=(128, 64)):
    """Five tokens, 4 / 2 heads of 64, bf16; strides in elements; positions or a tree: (code, text)."""
    pa = ge.load_package()
    cache = cache_at(pa, at)
    rc = pa.lib().ptoamd_kvcache_append_rope(ctypes.addressof(cache), at["out"], at["q"], 4, at["k"], at["v"], pa.BF16, 5, at["cu"], 3, at["table"], 10, 64, 0,
                                             at["positions"] if which == "positions" else None, at["tree"] if which == "tree" else None, int(which == "tree"), *q, *out, *k, *v,
                                             None)
    return rc, pa.lib().ptoamd_last_error().decode()


BYTES = {"table": 10 * 64 * 4, "positions": 20, "tree": 40, "cu": 12, "lengths": 8, "block_table": 16, "k_scale": 32, "v_scale": 32}
OUT = 5 * 256 * 2


@pytest.mark.parametrize("name", list(BYTES))
@pytest.mark.parametrize("end", ["first", "last"])
def test_append_over_what_it_reads(name, end):
    at = places()
    at["out"] = at[name] - OUT + 2 if end == "first" else at[name] + BYTES[name] - 2
    rc, error = append(at, "tree" if name == "tree" else "positions")
    assert rc == -1 and "q_out must not overlap" in error and (name in ("cu", "k_scale", "v_scale") or name in error), error


@pytest.mark.parametrize("by", [64, -64, 256, -256, 4 * 256, 1, -1])
def test_append_over_its_queries_but_in_place(by):
    at = places()
    rc, error = append({**at, "out": at["q"] + 2 * by}, "positions")
    assert rc == -1 and "q_out must be q or not overlap it" in error, error


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("by", [0, 64, -4 * 64 + 1, 127, 4 * 128 + 127])
def test_append_over_keys_or_values(name, by):
    at = places()
    rc, error = append({**at, "out": at[name] + 2 * by}, "positions")
    assert rc == -1 and "q_out must not overlap k or v" in error, error


@pytest.mark.parametrize("head", [3, 2, 7, -1])
def test_append_into_a_fused_product(head):
    """Queries, keys and values side by side, eight heads a token: results anywhere but over the queries themselves."""
    fused = AT + 100 * FAR
    at = places(q=fused, k=fused + 2 * 4 * 64, v=fused + 2 * 6 * 64, out=fused + 2 * 64 * head)
    strides = (512, 64)
    rc, error = append(at, "positions", strides, strides, strides, strides)
    assert rc == -1 and "overlap" in error, error


def keep(at):
    """Two sequences of eight drafted tokens, four entries each: (code, text)."""
    pa = ge.load_package()
    cache = cache_at(pa, at)
    rc = pa.lib().ptoamd_kvcache_keep(ctypes.addressof(cache), at["out"], at["q"], 4, at["cu"], 8, None)
    return rc, pa.lib().ptoamd_last_error().decode()


@pytest.mark.parametrize("name", ["block_table", "k_scale", "v_scale"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_new_lengths_over_what_keep_reads(name, end):
    at = places()
    rc, error = keep({**at, "out": at[name] - 4 if end == "first" else at[name] + BYTES[name] - 4})
    assert rc == -1 and "new_lengths must not overlap block_table or the scales" in error, error


@pytest.mark.parametrize("name", ["out", "lse"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_attention_over_its_tree(name, end):
    pa, at = ge.load_package(), places()
    cache = cache_at(pa, at)
    size = OUT if name == "out" else 5 * 4 * 4
    mine = {"out": at["out"], "lse": None, name: at["tree"] - size + 4 if end == "first" else at["tree"] + BYTES["tree"] - 4}
    rc = pa.lib().ptoamd_attention_kv8_tree(mine["out"], mine["lse"], ctypes.addressof(cache), at["tree"], 1, at["q"], pa.BF16, 4, 5, at["cu"], 3, 0, 256, 64, 256, 64, 0.125, 0,
                                            None, 0, None)
    error = pa.lib().ptoamd_last_error().decode()
    assert rc == -1 and "out and lse must not overlap the tree" in error, error
