"""What the operators around an 8-bit cache refuse, without a GPU: through the C ABI (the checks come before any launch) and through the package."""
import ctypes

import pytest
import torch

import __graft_entry__ as ge
from test_binding import outcome

NAMES = ["rope", "kvcache_append", "attention_kv8"]
BUF = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUF) + 255) // 256 * 256


def call(name, **change):
    """The entry point with good arguments but those changed (cache_...: a field of the cache): (code, text)."""
    pa = ge.load_package()
    cache = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, block_table=AT, lengths=AT, code_type=pa.I8, pages=4, kv_heads=2, page_size=16, head_dim=64, sequences=2,
                 max_pages=2, k_page_stride=2048, k_head_stride=1024, k_token_stride=64, v_page_stride=2048, v_head_stride=1024, v_token_stride=64)
    cache.update({k[6:]: v for k, v in change.items() if k.startswith("cache_")})
    good = {
        "ptoamd_rope_table": dict(table=AT, rows=10, rot=64, base=1e4, factor=1.0, low=0.0, high=0.0, magnitude=1.0, stream=None),
        "ptoamd_rope": dict(out=AT, x=AT, type=pa.BF16, table=AT, rows=10, positions=AT, tokens=2, heads=2, dim=64, rot=64, xt=128, xh=64, ot=128, oh=64,
                            interleaved=0, backward=0, stream=None),
        "ptoamd_kvcache_append": dict(cache=ctypes.addressof(pa._Kv8Cache(**cache)), k=AT, v=AT, type=pa.BF16, tokens=2, cu=None, most=1, kt=128, kh=64, vt=128,
                                      vh=64, stream=None),
        "ptoamd_attention_kv8": dict(out=AT, lse=None, cache=ctypes.addressof(pa._Kv8Cache(**cache)), q=AT, type=pa.BF16, heads=4, tokens=2, cu=None, most=1,
                                     max_length=0, qt=256, qh=64, ot=256, oh=64, scale=0.125, causal=1, window=0, workspace=None, bytes=0, stream=None),
    }[name]
    unknown = {k for k in change if not k.startswith("cache_")} - set(good)
    assert not unknown, unknown
    keep = pa._Kv8Cache(**cache)
    if "cache" in good:
        good["cache"] = ctypes.addressof(keep)
    good.update({k: v for k, v in change.items() if not k.startswith("cache_")})
    rc = getattr(pa.lib(), name)(*good.values())
    return rc, pa.lib().ptoamd_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(table=None), -1, "null"), (dict(rows=0), -1, "positive"), (dict(rot=63), -1, "even"), (dict(rot=0), -1, "positive"), (dict(base=0.0), -1, "positive"),
    (dict(factor=float("nan")), -1, "positive"), (dict(low=2.0, high=1.0), -1, "ramp_low"), (dict(magnitude=float("inf")), -1, "finite")])
def test_rope_table(change, code, text):
    rc, error = call("ptoamd_rope_table", **change)
    assert rc == code and text in error


@pytest.mark.parametrize("change,code,text", [
    (dict(out=None), -1, "null"), (dict(positions=None), -1, "null"), (dict(tokens=-1), -1, "negative"), (dict(heads=0), -1, "positive"), (dict(rows=0), -1, "positive"),
    (dict(rot=66), -1, "rot_dim"), (dict(rot=31), -1, "even"), (dict(type=3), -2, "f32, f16 or bf16"), (dict(x=AT + 1), -3, "aligned"),
    (dict(ot=64), -1, "in place"), (dict(heads=1 << 20), -2, "too many")])
def test_rope(change, code, text):
    rc, error = call("ptoamd_rope", **change)
    assert rc == code and text in error
    assert call("ptoamd_rope", tokens=0)[0] == 0


CACHE = [(dict(cache=None), -1, "null cache"), (dict(cache_code_type=1), -2, "int8 or E4M3"), (dict(cache_pages=0), -1, "positive"), (dict(cache_sequences=0), -1, "positive"),
         (dict(cache_page_size=48), -2, "page_size"), (dict(cache_page_size=8), -2, "page_size"), (dict(cache_max_pages=1 << 30), -2, "too many"),
         (dict(cache_k=None), -1, "null"), (dict(cache_lengths=None), -1, "null"), (dict(cache_v=AT + 4), -3, "multiples of 8"), (dict(cache_k_token_stride=60), -3, "multiples of 8"),
         (dict(tokens=-1), -1, "negative"), (dict(tokens=3), -1, "sequences * max_tokens"), (dict(most=2), -1, "sequences * max_tokens"), (dict(cache_head_dim=60), -2, "multiple of 8"),
         (dict(cache_head_dim=520), -2, "at most 512"), (dict(cache_kv_heads=70000), -2, "65535")]


@pytest.mark.parametrize("change,code,text", CACHE + [(dict(k=None), -1, "null"), (dict(type=4), -2, "f32, f16 or bf16"), (dict(v=AT + 1), -3, "aligned")])
def test_append(change, code, text):
    rc, error = call("ptoamd_kvcache_append", **change)
    assert rc == code and text in error, error
    assert call("ptoamd_kvcache_append", tokens=0, most=0)[0] == 0


@pytest.mark.parametrize("change,code,text", [c for c in CACHE if "cache_kv_heads" not in c[0]] + [
    (dict(q=None), -1, "null"), (dict(out=None), -1, "null"), (dict(type=0), -2, "f16 or bf16"), (dict(heads=3), -1, "multiple of kv_heads"), (dict(heads=0), -1, "multiple of kv_heads"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(window=-1), -1, "window"),
    (dict(max_length=-1), -1, "max_length"), (dict(q=AT + 1), -3, "aligned"), (dict(lse=AT + 2), -3, "aligned")])
def test_attention(change, code, text):
    rc, error = call("ptoamd_attention_kv8", **change)
    assert rc == code and text in error, error
    assert call("ptoamd_attention_kv8", tokens=0, most=0)[0] == 0


@pytest.mark.parametrize("name", NAMES)
def test_the_package_raises_with_a_reason(name):
    pa = ge.load_package()
    t = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)  # noqa: E731
    cache = (t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, dtype=torch.float32), t(4, 2, dtype=torch.float32),
             t(2, 2, dtype=torch.int32), t(2, dtype=torch.int32), pa.I8)
    args = {"rope": (t(2, 2, 64), t(10, 64, dtype=torch.float32), t(2, dtype=torch.int32)), "kvcache_append": (t(2, 2, 64), t(2, 2, 64)) + cache,
            "attention_kv8": (t(2, 4, 64),) + cache}[name]
    with pytest.raises(pa.PtoAmdError, match="device tensor"):
        getattr(pa, name)(*args)  # (host tensors)
    with pytest.raises(pa.PtoAmdError, match=r"\[tokens"):
        getattr(pa, name)(args[0][0], *args[1:])
    with pytest.raises(pa.PtoAmdError, match="f16"):
        getattr(pa, name)(args[0].double(), *args[1:])


@pytest.mark.parametrize("name", NAMES)
def test_the_native_form_refuses_like_the_function(name):
    import copy
    import inspect
    import pickle

    f = getattr(ge.load_package(), name)
    assert f is not f.__wrapped__ and inspect.signature(f) == inspect.signature(f.__wrapped__) and f.__doc__ == f.__wrapped__.__doc__
    assert copy.copy(f) is f and pickle.loads(pickle.dumps(f)) is f
    a, v = torch.zeros(4, 2, 64), torch.zeros(4)
    calls = [((), {}), ((a,), {}), ((a, a, a), {"wrong": 1}), ((a, v, v), {}), ((a,) * 30, {}), ((a,) * 9, {}), ((a.half(),) * 9, {}), ((1, 2, 3, 4, 5, 6, 7, 8, 9), {}),
             ((None,) * 9, {}), ((a, a, a), {"x": a})]
    for args, kw in calls:
        assert outcome(f, *args, **kw) == outcome(f.__wrapped__, *args, **kw), (name, args, kw)
