"""What the operators around drafted trees refuse, without a GPU: through the C ABI (the checks come before any launch) and through the package."""
import ctypes
import inspect

import pytest
import torch

import __graft_entry__ as ge
from test_binding import outcome
from test_kv8_refusals import AT
from test_kv8_refusals import CACHE as KV8

NAMES = ["draft_tree", "kvcache_append_rope", "attention_kv8_tree", "kvcache_keep"]


def call(name, **change):
    """The entry point with good arguments but those changed (cache_...: a field of the cache): (code, text)."""
    pa = ge.load_package()
    cache = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, block_table=AT, lengths=AT, code_type=pa.I8, pages=4, kv_heads=2, page_size=16, head_dim=64, sequences=2,
                 max_pages=2, k_page_stride=2048, k_head_stride=1024, k_token_stride=64, v_page_stride=2048, v_head_stride=1024, v_token_stride=64)
    cache.update({k[6:]: v for k, v in change.items() if k.startswith("cache_")})
    keep = pa._Kv8Cache(**cache)
    c = ctypes.addressof(keep)
    good = {
        "ptoamd_draft_tree": dict(tree=AT, words=1, parents=AT, tokens=2, sequences=2, cu=None, most=1, stream=None),
        "ptoamd_kvcache_append_rope": dict(cache=c, q_out=AT, q=AT, heads=4, k=AT, v=AT, type=pa.BF16, tokens=2, cu=None, most=1, table=AT, rows=10, rot=64,
                                           interleaved=0, positions=None, tree=None, words=0, qt=256, qh=64, ot=256, oh=64, kt=128, kh=64, vt=128, vh=64, stream=None),
        "ptoamd_attention_kv8_tree": dict(out=AT, lse=None, cache=c, tree=AT, words=1, q=AT, type=pa.BF16, heads=4, tokens=2, cu=None, most=1, max_length=0, qt=256,
                                          qh=64, ot=256, oh=64, scale=0.125, window=0, workspace=None, bytes=0, stream=None),
        "ptoamd_kvcache_keep": dict(cache=c, new=AT + 1024, kept=AT, max_kept=4, cu=None, most=8, stream=None),
    }[name]
    fields = {k: v for k, v in change.items() if not k.startswith("cache_")}
    assert not set(fields) - set(good), fields
    good.update(fields)
    rc = getattr(pa.lib(), name)(*good.values())
    return rc, pa.lib().ptoamd_last_error().decode()


TREE = [(dict(words=0), -1, "words"), (dict(words=5), -1, "words"), (dict(cu=AT, tokens=70, most=65), -1, "words"),
        (dict(cu=AT, tokens=300, most=257, words=4), -2, "at most 256"), (dict(tree=AT + 4), -3, "aligned")]


@pytest.mark.parametrize("change,code,text", TREE + [
    (dict(tree=None), -1, "null"), (dict(parents=None), -1, "null"), (dict(parents=AT + 2), -3, "aligned"), (dict(tokens=-1), -1, "negative"),
    (dict(sequences=0), -1, "positive"), (dict(most=-1), -1, "negative"), (dict(tokens=3), -1, "sequences * max_tokens"),
    (dict(parents=AT + 8), -1, "overlap"), (dict(parents=AT - 4), -1, "overlap"), (dict(parents=AT + 64, cu=AT - 8), -1, "overlap")])
def test_draft_tree(change, code, text):
    rc, error = call("ptoamd_draft_tree", **change)
    assert rc == code and text in error, error
    assert call("ptoamd_draft_tree", tokens=0, most=0)[0] == 0


@pytest.mark.parametrize("change,code,text", KV8 + [
    (dict(k=None), -1, "null"), (dict(q=None), -1, "null"), (dict(q_out=None), -1, "null"), (dict(table=None), -1, "null"), (dict(type=4), -2, "f32, f16 or bf16"),
    (dict(v=AT + 1), -3, "aligned"), (dict(q=AT + 1), -3, "aligned"), (dict(table=AT + 2), -3, "aligned"), (dict(positions=AT + 1), -3, "aligned"),
    (dict(rows=0), -1, "positive"), (dict(heads=-1), -1, "negative"), (dict(heads=1 << 20), -2, "too many"), (dict(rot=66), -1, "rot_dim"), (dict(rot=31), -1, "even"),
    (dict(rot=0), -1, "even"), (dict(ot=64), -1, "in place"), (dict(positions=AT, tree=AT, words=1), -1, "not both")]
    + [({"tree": AT, "words": 1, **c}, code, text) for c, code, text in TREE])
def test_append_rope(change, code, text):
    rc, error = call("ptoamd_kvcache_append_rope", **change)
    assert rc == code and text in error, error
    assert call("ptoamd_kvcache_append_rope", tokens=0, most=0)[0] == 0


@pytest.mark.parametrize("change,code,text", [c for c in KV8 if "cache_kv_heads" not in c[0]] + TREE + [
    (dict(tree=None), -1, "null"), (dict(q=None), -1, "null"), (dict(out=None), -1, "null"), (dict(type=0), -2, "f16 or bf16"), (dict(heads=3), -1, "multiple of kv_heads"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(window=-1), -1, "window"), (dict(max_length=-1), -1, "max_length"),
    (dict(q=AT + 1), -3, "aligned"), (dict(lse=AT + 2), -3, "aligned"), (dict(cu=AT, tokens=70, most=60, window=59), -2, "window"),
    (dict(cu=AT, tokens=50, most=60, window=49), -2, "window")])
def test_attention(change, code, text):
    rc, error = call("ptoamd_attention_kv8_tree", **change)
    assert rc == code and text in error, error
    assert call("ptoamd_attention_kv8_tree", tokens=0, most=0)[0] == 0


@pytest.mark.parametrize("change,code,text", [c for c in KV8 if not {"tokens", "most"} & set(c[0])] + [
    (dict(new=None), -1, "null"), (dict(kept=None), -1, "null"), (dict(kept=AT + 2), -3, "aligned"), (dict(new=AT + 1026), -3, "aligned"), (dict(most=0), -1, "positive"),
    (dict(max_kept=-1), -1, "negative"), (dict(most=257), -2, "at most 256"), (dict(new=AT), -1, "must not be lengths"), (dict(new=AT + 4), -1, "must not be lengths"),
    (dict(new=AT - 4), -1, "must not be lengths"), (dict(new=AT + 28, cache_lengths=AT + 1024), -1, "overlap kept"), (dict(kept=AT + 1020), -1, "overlap kept"),
    (dict(cu=AT + 1016), -1, "overlap kept or cu_tokens")])
def test_keep(change, code, text):
    rc, error = call("ptoamd_kvcache_keep", **change)
    assert rc == code and text in error, error


def arguments(pa):
    t = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)  # noqa: E731
    cache = (t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, dtype=torch.float32), t(4, 2, dtype=torch.float32),
             t(2, 2, dtype=torch.int32), t(2, dtype=torch.int32), pa.I8)
    return {"draft_tree": (t(2, dtype=torch.int32), 2), "kvcache_append_rope": (t(2, 4, 64), t(2, 2, 64), t(2, 2, 64)) + cache + (t(10, 64, dtype=torch.float32),),
            "attention_kv8_tree": (t(2, 4, 64),) + cache + (t(2, 1, dtype=torch.int64),), "kvcache_keep": (t(2, 3, dtype=torch.int32),) + cache}


@pytest.mark.parametrize("name", NAMES)
def test_the_package_raises_with_a_reason(name):
    pa = ge.load_package()
    args = arguments(pa)[name]
    with pytest.raises(pa.PtoAmdError, match="device tensor"):
        getattr(pa, name)(*args, **({"max_tokens": 4} if name == "kvcache_keep" else {}))  # (host tensors)
    if name == "kvcache_keep":
        with pytest.raises(pa.PtoAmdError):
            getattr(pa, name)(*args)


@pytest.mark.parametrize("name", NAMES)
def test_the_native_form_refuses_like_the_function(name):
    import copy
    import pickle

    f = getattr(ge.load_package(), name)
    assert f is not f.__wrapped__ and inspect.signature(f) == inspect.signature(f.__wrapped__) and f.__doc__ == f.__wrapped__.__doc__
    assert copy.copy(f) is f and pickle.loads(pickle.dumps(f)) is f
    a, v = torch.zeros(4, 2, 64), torch.zeros(4)
    args = arguments(ge.load_package())[name]
    calls = [((), {}), ((a,), {}), ((a, a, a), {"wrong": 1}), ((a, v, v), {}), ((a,) * 30, {}), ((a,) * 9, {}), ((a.half(),) * 12, {}), (tuple(range(12)), {}),
             ((None,) * 12, {}), ((a, a, a), {"x": a}), (args, {}), (args[:-1], {}), (args, {"max_tokens": 1}), (args, {"max_tokens": None})]
    for args, kw in calls:
        assert outcome(f, *args, **kw) == outcome(f.__wrapped__, *args, **kw), (name, args, kw)
