"""The work that the operators around the cache are measured on: rotary positions, the append of new keys and values to a
cache held in 8 bits, and attention over that cache.

  rope       queries and keys of a fused QKV product turned by their positions (or their gradients turned back): half and
             interleaved pairs, the whole head or its first part, f32, f16 and bf16
  append     keys and values of new tokens quantised into the pages of a cache with a scale for each page and head: one token
             of many sequences (decode), whole prompts (prefill); int8 and E4M3 codes
  attention  queries of one token, of a few (several tokens guessed ahead), of a chunk or a whole prompt over such a cache,
             with shared heads, causal, with and without a window

``own`` false: the plain forms, in elementary torch operations; true: the package's entry points.
"""
import importlib
import math
import random

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_LARGEST = {"i8": 127.0, "e4m3": 448.0}
_TINY = 2.0 ** -126  # a smaller scale counts as zero
_DEV = "cuda"


# ---- cases ----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 16 sequences: 64 query and 8 key heads of the fused product, each token at a position of its own
        dict(name="rope_decode_16", kind="rope", dtype="bf16", tokens=16, heads=72, other=8, dim=128, rot=128, interleaved=False,
             backward=False, factor=1.0, longest=32768),
        # a prefill batch of a long-context model (frequencies scaled): 32 query and 8 key heads
        dict(name="rope_prefill_8192", kind="rope", dtype="bf16", tokens=8192, heads=40, other=8, dim=128, rot=128, interleaved=False,
             backward=False, factor=8.0, longest=131072),
        # the gradient of a rotation of the first 32 of 80 elements, interleaved pairs, f32, odd counts of tokens and heads
        dict(name="rope_partial_gradient", kind="rope", dtype="f32", tokens=2003, heads=33, other=0, dim=80, rot=32, interleaved=True,
             backward=True, factor=1.0, longest=4096),
        # a decode step of 48 sequences: one token each goes into a page that mostly holds older ones
        dict(name="append_decode_48", kind="append", dtype="bf16", code="i8", seqs=48, tokens=1, ragged=False, longest=8192, heads=8,
             dim=128, page=64, spread=3),
        # prompts of seven sequences, their lengths and their starts in the cache ragged
        dict(name="append_prefill_ragged", kind="append", dtype="bf16", code="e4m3", seqs=7, tokens=2048, ragged=True, longest=8192,
             heads=8, dim=128, page=32, spread=4),
        # one short sequence: the call is launches and little else
        dict(name="attn_decode_1x300", kind="attention", dtype="bf16", code="i8", seqs=1, tokens=1, ragged=False, longest=300,
             lengths="same", heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0, lse=False, spread=1),
        # a decode step of 16 sequences of 8192 tokens, eight queries to a key head
        dict(name="attn_decode_16x8192", kind="attention", dtype="bf16", code="e4m3", seqs=16, tokens=1, ragged=False, longest=8192,
             lengths="same", heads=64, kv_heads=8, dim=128, page=64, causal=True, window=0, lse=False, spread=1),
        # one very long sequence: a single row of work per head that has to fill the card
        dict(name="attn_decode_1x131072", kind="attention", dtype="bf16", code="i8", seqs=1, tokens=1, ragged=False, longest=131072,
             lengths="same", heads=64, kv_heads=8, dim=128, page=64, causal=True, window=0, lse=False, spread=1),
        # 48 sequences of very different lengths, a key head to every query head, with the log-sums that joins need
        dict(name="attn_decode_48_ragged", kind="attention", dtype="f16", code="e4m3", seqs=48, tokens=1, ragged=False, longest=4001,
             lengths="ragged", heads=16, kv_heads=16, dim=64, page=16, causal=True, window=0, lse=True, spread=7),
        # five tokens guessed ahead for eight sequences, heads of 256 elements, a sliding window
        dict(name="attn_guess_8x5_window", kind="attention", dtype="bf16", code="i8", seqs=8, tokens=5, ragged=False, longest=6000,
             lengths="ragged", heads=16, kv_heads=2, dim=256, page=64, causal=True, window=1024, lse=False, spread=5),
        # chunks of prompts over long caches, ragged: 3 sequences of up to 512 new tokens
        dict(name="attn_chunk_3x512", kind="attention", dtype="bf16", code="i8", seqs=3, tokens=512, ragged=True, longest=16384,
             lengths="ragged", heads=32, kv_heads=8, dim=128, page=32, causal=True, window=0, lse=False, spread=6),
        # a whole prompt: the largest product
        dict(name="attn_prefill_8192", kind="attention", dtype="bf16", code="e4m3", seqs=1, tokens=8192, ragged=False, longest=8192,
             lengths="same", heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0, lse=False, spread=1),
    ]


def _between(rng, lo, hi, multiple=1):
    """An integer of [lo, hi], spread over its logarithm, on the given multiple."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(v / multiple + 0.5) * multiple))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "attention"])
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        return dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16", "bf16"]), tokens=_between(rng, 1, 8192), heads=_between(rng, 1, 72),
                    other=rng.choice([0, 1, 8]), dim=dim, rot=rng.choice([dim, dim, dim // 2, 32]), interleaved=rng.random() < 0.4,
                    backward=rng.random() < 0.4, factor=rng.choice([1.0, 4.0, 8.0]), longest=_between(rng, 4096, 131072))
    while True:
        page, dim, code = rng.choice([16, 32, 64, 128]), rng.choice([64, 128, 128, 256]), rng.choice(["i8", "e4m3"])
        common = dict(code=code, dim=dim, page=page, spread=rng.randrange(1, 1000))
        if kind == "append":
            case = dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16", "bf16"]), seqs=_between(rng, 1, 64),
                        tokens=rng.choice([1, 1, _between(rng, 2, 4096)]), ragged=rng.random() < 0.6, longest=_between(rng, 4096, 16384),
                        heads=rng.choice([1, 2, 4, 8, 16]), **common)
            if case["seqs"] * case["longest"] * case["heads"] * dim <= 1 << 27 and case["seqs"] * case["tokens"] <= 32768:
                return case
            continue
        kv = rng.choice([1, 2, 4, 8, 16])
        tokens = rng.choice([1, 1, 1, rng.randrange(2, 9), _between(rng, 9, 4096)])
        case = dict(kind=kind, dtype=rng.choice(["f16", "bf16", "bf16"]), seqs=_between(rng, 1, 64), tokens=tokens, ragged=tokens > 8 and rng.random() < 0.7,
                    longest=_between(rng, max(64, tokens), 65536), lengths=rng.choice(["same", "ragged"]), heads=kv * rng.choice([1, 2, 4, 7, 8]),
                    kv_heads=kv, causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, _between(rng, 64, 4096)]), lse=rng.random() < 0.3, **common)
        if case["seqs"] * case["longest"] * kv * dim <= 1 << 27 and case["seqs"] * case["longest"] * tokens * case["heads"] * dim <= 1 << 36:
            return case


def _lengths(case):
    """Tokens new to each sequence, and its length with them."""
    rng = random.Random(case["spread"])
    new, total = [], []
    for _ in range(case["seqs"]):
        n = rng.randint(max(1, case["tokens"] // 4), case["tokens"]) if case["ragged"] else case["tokens"]
        if case["kind"] == "append":
            length = rng.randint(n, case["longest"])
        elif case["lengths"] == "same":
            length = case["longest"]
        else:
            length = max(n, int(math.exp(rng.uniform(math.log(max(1, case["longest"] // 256)), math.log(case["longest"])))))
        new.append(n)
        total.append(length)
    if case["ragged"]:
        new[-1], total[-1] = case["tokens"], max(case["tokens"], total[-1])
    return new, total


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _frequencies(case):
    """Of each pair, in 64 bits: scaled by ``factor`` for the slow ones, a ramp between (what long-context models do)."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=_DEV)
    f = 10000.0 ** (-2.0 * i / case["rot"])
    ramp = ((i - case["rot"] / 8) / (case["rot"] / 4)).clamp(0, 1) if case["factor"] != 1.0 else torch.zeros_like(i)
    return f * (1 - ramp) + f / case["factor"] * ramp


def _values(gen, shape, dtype, heads_at, spread):
    """Activations: normal, with a few channels of a head larger than the others, as keys have them."""
    x = torch.randn(shape, generator=gen, device=_DEV, dtype=torch.float32)
    channel = torch.exp(spread * torch.randn((shape[heads_at], shape[-1]), generator=gen, device=_DEV))
    view = [1] * len(shape)
    view[heads_at], view[-1] = shape[heads_at], shape[-1]
    return x.mul_(channel.view(view)).to(dtype)


def _round(x, code):
    """Values in units of their scale -> codes."""
    return x.round().clamp(-127, 127).to(torch.int8) if code == "i8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(gen, pages, case, heads, spread):
    """A cache that holds something everywhere: codes [pages, heads, page, dim] and scales [pages, heads]."""
    x = _values(gen, (pages, heads, case["page"], case["dim"]), torch.float32, 1, spread)
    x.mul_(torch.exp(0.2 * torch.randn((pages, heads, 1, 1), generator=gen, device=_DEV)))
    scale = x.abs().amax(dim=(2, 3)) / _LARGEST[case["code"]]
    return _round(x.div_(scale[:, :, None, None]), case["code"]), scale


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "rope":
        qkv = _values(gen, (case["tokens"], case["heads"] + case["other"], case["dim"]), _DTYPE[case["dtype"]], 1, 0.3)
        s["x"] = qkv[:, :case["heads"]]
        s["positions"] = torch.randint(0, case["longest"], (case["tokens"],), generator=gen, device=_DEV, dtype=torch.int32)
        angle = torch.arange(case["longest"], dtype=torch.float64, device=_DEV)[:, None] * _frequencies(case)
        s["table"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        return s
    new, total = _lengths(case)
    heads = case["heads"] if case["kind"] == "append" else case["kv_heads"]
    wide = -(-max(total) // case["page"])
    pages = case["seqs"] * wide + 3
    s["k_cache"], s["k_scale"] = _cache(gen, pages, case, heads, 0.4)
    s["v_cache"], s["v_scale"] = _cache(gen, pages, case, heads, 0.1)
    s["block_table"] = torch.randperm(pages, generator=gen, device=_DEV)[:case["seqs"] * wide].view(case["seqs"], wide).to(torch.int32)
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device=_DEV)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=_DEV)
    s["max_tokens"], s["max_length"] = max(new), max(total)
    count, dtype = starts[-1], _DTYPE[case["dtype"]]
    if case["kind"] == "append":
        s["k"] = _values(gen, (count, heads, case["dim"]), dtype, 1, 0.4)
        s["v"] = _values(gen, (count, heads, case["dim"]), dtype, 1, 0.1)
    else:  # queries lie beside the keys that were turned with them
        s["q"] = _values(gen, (count, case["heads"] + heads, case["dim"]), dtype, 1, 0.2)[:, :case["heads"]]
        s["scale"] = case["dim"] ** -0.5
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "append": _own_append, "attention": _own_attention}[kind](state)
    return {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[kind](state)


def _package():
    return importlib.import_module("pto-isa-mirror_amd")


def _own_rope(s):
    c = s["case"]
    return _package().rope(s["x"], s["table"], s["positions"], interleaved=c["interleaved"], backward=c["backward"])


def _own_append(s):
    pa, c = _package(), s["case"]
    ragged = s["starts"] if c["ragged"] else None
    pa.kvcache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["lengths"],
                      pa.I8 if c["code"] == "i8" else pa.E4M3, cu_tokens=ragged, max_tokens=s["max_tokens"])
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attention(s):
    pa, c = _package(), s["case"]
    ragged = s["starts"] if c["ragged"] else None
    return pa.attention_kv8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["lengths"],
                            pa.I8 if c["code"] == "i8" else pa.E4M3, cu_tokens=ragged, max_tokens=s["max_tokens"], max_length=s["max_length"],
                            scale=s["scale"], causal=c["causal"], window=c["window"], want_lse=c["lse"])


def _plain_rope(s):
    c, x = s["case"], s["x"].float()
    half = c["rot"] // 2
    turn = s["table"][s["positions"].long()]
    cos, sin = turn[:, None, :half], turn[:, None, half:]
    if c["backward"]:
        sin = -sin
    if c["interleaved"]:
        a, b = x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(2)
    else:
        a, b = x[..., :half], x[..., half:c["rot"]]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., c["rot"]:]], dim=-1).to(s["x"].dtype)


def _token_places(s, count):
    """Of every new token: its sequence and its place in it."""
    at = torch.arange(count, device=_DEV)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), at, right=True)
    old = s["lengths"].long() - (s["starts"][1:] - s["starts"][:-1]).long()
    return seq, at - s["starts"][seq].long(), old


def _plain_append(s):
    c = s["case"]
    seq, nth, old = _token_places(s, s["k"].shape[0])
    place = old[seq] + nth
    page = s["block_table"][seq, place // c["page"]].long()
    slot = place % c["page"]
    last = (old // c["page"]).clamp(max=s["block_table"].shape[1] - 1)
    partial = s["block_table"].gather(1, last[:, None])[:, 0].long()  # the page of each sequence that may hold older tokens
    held = (old - last * c["page"]).clamp(0, c["page"])
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.float()
        largest = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, scales.shape[1]), x.abs().amax(dim=2), "amax")
        kept = torch.zeros_like(scales)
        kept[partial] = scales[partial] * (held > 0)[:, None]
        grown = torch.maximum(kept, largest / _LARGEST[c["code"]])
        grown = torch.where(grown < _TINY, 0.0, grown)
        before, after = kept[partial], grown[partial]
        ratio = torch.where(after > before, before / after, 1.0)
        raw = codes.view(torch.uint8)
        older = _round(raw[partial].view(codes.dtype).float() * ratio[:, :, None, None], c["code"]).view(torch.uint8)
        is_older = torch.arange(c["page"], device=_DEV)[None, :] < held[:, None]
        raw[partial] = torch.where(is_older[:, None, :, None], older, raw[partial])
        touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=_DEV)
        touched[page] = True
        scales.copy_(torch.where(touched[:, None], grown, scales))
        unit = grown[page]
        inverse = torch.where(unit > 0, torch.ones_like(unit) / unit, 0.0)
        raw[page, :, slot] = _round(x * inverse[:, :, None], c["code"]).view(torch.uint8)
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    c = s["case"]
    kv, group, dim = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    most = s["max_tokens"]
    seqs, count = c["seqs"], s["q"].shape[0]
    n = (s["starts"][1:] - s["starts"][:-1]).long()
    nth = torch.arange(most, device=_DEV)
    rows = (s["starts"][:-1].long()[:, None] + nth).clamp(max=count - 1)
    q = s["q"].float()[rows].view(seqs, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, dim)
    table = s["block_table"].long()
    k, v = ((codes.view(torch.uint8)[table].view(codes.dtype).float() * scales[table][..., None, None]).transpose(1, 2).reshape(seqs, kv, -1, dim)
            for codes, scales in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
    score = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(seqs, kv, most, group, -1)
    key = torch.arange(score.shape[-1], device=_DEV)
    at = (s["lengths"].long() - n)[:, None] + nth  # the place of each query
    seen = key < s["lengths"][:, None, None]
    if c["causal"]:
        seen = seen & (key <= at[:, :, None])
    if c["window"]:
        seen = seen & (key > at[:, :, None] - c["window"])
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.view(seqs, kv, most * group, -1), v).view(seqs, kv, most, group, dim) / torch.where(total > 0, total, 1.0)
    seq, place, _ = _token_places(s, count)
    out = out.permute(0, 2, 1, 3, 4).reshape(seqs, most, c["heads"], dim)[seq, place].to(s["q"].dtype)
    if not c["lse"]:
        return out
    return out, (top + total.log()).permute(0, 2, 1, 3, 4).reshape(seqs, most, c["heads"])[seq, place]


# ---- the same by definition, in 64 bits ---------------------------------------------------------------------------------

def _grid_e4m3(x):
    """The nearest value that E4M3 holds (four significant bits, 2^-9 the smallest, 448 the largest), ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_rope(case, s):
    x = s["x"].double()
    angle = s["positions"].double()[:, None] * _frequencies(case)
    turn = torch.polar(torch.ones_like(angle), -angle if case["backward"] else angle)[:, None]
    half, rot = case["rot"] // 2, case["rot"]
    pair = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else torch.complex(x[..., :half], x[..., half:rot])
    pair = pair * turn
    out = x.clone()
    if case["interleaved"]:
        out[..., 0:rot:2], out[..., 1:rot:2] = pair.real, pair.imag
    else:
        out[..., :half], out[..., half:rot] = pair.real, pair.imag
    return out


def _exact_append(case, s):
    new, total = _lengths(case)
    size, got = case["page"], {}
    table, starts = s["block_table"].tolist(), s["starts"].tolist()
    for name in ("k", "v"):
        codes, scales, x = s[name + "_cache"].double(), s[name + "_scale"].double(), s[name].double()
        for q in range(case["seqs"]):
            first = total[q] - new[q]
            for block in range(first // size, -(-total[q] // size)):
                lo, hi = max(first, block * size), min(total[q], (block + 1) * size)
                rows = x[starts[q] + lo - first:starts[q] + hi - first].transpose(0, 1)  # [heads, tokens, dim]
                unit = rows.abs().amax(dim=(1, 2)) / _LARGEST[case["code"]]
                page, older = table[q][block], lo - block * size
                if older:
                    unit = torch.maximum(unit, scales[page])
                    if case["code"] == "e4m3":
                        codes[page, :, :older] = _grid_e4m3(codes[page, :, :older] * (scales[page] / unit)[:, None, None])
                scales[page] = unit
                if case["code"] == "e4m3":
                    codes[page, :, older:older + hi - lo] = _grid_e4m3(rows / unit[:, None, None])
        # int8 codes are whole numbers, compared as such
        got[name], got[name + "_scale"] = codes if case["code"] == "e4m3" else None, scales
    return got


def _exact_attention(case, s):
    new, total = _lengths(case)
    group, starts = case["heads"] // case["kv_heads"], s["starts"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=_DEV)
    for q in range(case["seqs"]):
        pages = s["block_table"][q, :-(-total[q] // case["page"])].long()
        for h in range(case["heads"]):
            j = h // group
            k, v = ((s[x + "_cache"][pages, j].double() * s[x + "_scale"][pages, j].double()[:, None, None]).flatten(0, 1)[:total[q]] for x in "kv")
            for lo in range(0, new[q], 2048):
                hi = min(new[q], lo + 2048)
                place = torch.arange(lo, hi, device=_DEV) + (total[q] - new[q])
                key = torch.arange(total[q], device=_DEV)
                hidden = torch.zeros((hi - lo, total[q]), dtype=torch.bool, device=_DEV)
                if case["causal"]:
                    hidden |= key[None] > place[:, None]
                if case["window"]:
                    hidden |= key[None] <= place[:, None] - case["window"]
                logit = (s["q"][starts[q] + lo:starts[q] + hi, h].double() @ k.t()) * s["scale"]
                logit[hidden] = -math.inf
                norm = torch.logsumexp(logit, dim=1)
                weight = torch.nan_to_num(torch.exp(logit - norm[:, None]), nan=0.0)
                out[starts[q] + lo:starts[q] + hi, h] = weight @ v
                lse[starts[q] + lo:starts[q] + hi, h] = norm
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attention": _exact_attention}[case["kind"]](case, s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * _SIZE[case["dtype"]] + case["tokens"] * (4 * case["rot"] + 4), "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    new, total = _lengths(case)
    if case["kind"] == "append":  # (older codes are counted as not touched: they change only where a scale grows)
        values = 2 * sum(new) * case["heads"] * case["dim"]
        blocks = sum(-(-t // case["page"]) - (t - n) // case["page"] for n, t in zip(new, total))
        return {"bytes": values * (_SIZE[case["dtype"]] + 1) + blocks * (16 * case["heads"] + 4) + 4 * case["seqs"], "flops": 3 * values}
    seen, pairs = 0, 0
    for n, t in zip(new, total):
        first = max(0, t - n + 1 - case["window"]) if case["window"] else 0
        seen += t - first
        if case["causal"] or case["window"]:
            at = range(t - n, t)
            pairs += sum((p + 1 if case["causal"] else t) - (max(0, p + 1 - case["window"]) if case["window"] else 0) for p in at)
        else:
            pairs += n * t
    blocks = seen / case["page"]
    return {"bytes": 2 * _SIZE[case["dtype"]] * sum(new) * case["heads"] * case["dim"] + 2 * seen * case["kv_heads"] * case["dim"] +
            blocks * (8 * case["kv_heads"] + 4) + (4 * sum(new) * case["heads"] if case["lse"] else 0),
            "flops": 4 * case["dim"] * case["heads"] * pairs}
