"""Drafted trees over an 8-bit cache by their definitions, in 64 bits.  (How far attention may be off: kv8_reference.check_attention.)"""
import math
import random

import torch


def parents_of(counts, seed, width=0):
    """Of every sequence's tokens: any drafted before it, or -1; width: among that many before it (deep trees)."""
    rng = random.Random(seed)
    return [[rng.randrange(max(-1, i - width) if width else -1, i) for i in range(n)] for n in counts]


def ways_of(parents):
    """Of every sequence's tokens: the set of those that it sees.  A parent that is neither -1 nor before the token: none."""
    ways = []
    for mine in parents:
        w = []
        for i, p in enumerate(mine):
            w.append(frozenset() if p < -1 or p >= i else (w[p] if p >= 0 else frozenset()) | {i})
        ways.append(w)
    return ways


def rows_of(ways, words):
    """Sets as rows of 64-bit words [tokens, words]."""
    rows = []
    for way in (w for mine in ways for w in mine):
        bits = sum(1 << t for t in way)
        rows.append([(bits >> (64 * w) & (2 ** 64 - 1)) - (2 ** 64 if bits >> (64 * w + 63) & 1 else 0) for w in range(words)])
    return torch.tensor(rows, dtype=torch.int64, device="cuda").view(-1, words)


def flat(parents):
    return torch.tensor([p for mine in parents for p in mine], dtype=torch.int32, device="cuda")


def attention(q, cache, ways, window=0, scale=None):
    """As kv8_reference.attention, of drafted tokens: (out, lse, magnitude, spread) in 64 bits."""
    return attention_and_least(q, cache, ways, window, scale)[0]


def attention_and_least(q, cache, ways, window=0, scale=None):
    """That, and what results may be off by beside it where elements of the keys of large weights are small.
    A weight (p times its page's value scale s) is f16 on a scale on which the largest p s of the row is 2^11 or more; steps of f16 end at 2^-24, so a
    rounding is off by 2^-25 at most where it is not relative: 2^-36 of the largest p s, times the code of each key.
    An int8 code c is multiplied as c + 128, and 128 times the weights taken off in the same tile: sums on the way are up to 255 times the weights', whatever
    the codes, and each instruction rounds them to f32 up to eight times (its 32 products are added four at a time): 16 * 255 * 2^-24 < 2^-12 of the sum of
    p s."""
    tokens, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    least = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    spread = torch.zeros((tokens, heads), dtype=torch.float64, device="cuda")
    at = 0
    for s, mine in enumerate(ways):
        n, length = len(mine), int(cache.lengths[s])
        if n and length:
            old = length - n
            seen = torch.zeros((n, length), dtype=torch.bool)
            for i, way in enumerate(mine):
                first = max(0, old + len(way - {i}) - window + 1) if window else 0
                seen[i, min(first, max(old, 0)):max(old, 0)] = True
                for t in way:
                    if 0 <= t < n and old + t >= 0:
                        seen[i, old + t] = True
            seen = seen.cuda()
            group = heads // cache.kv_heads
            k, v = (x[s].repeat_interleave(group, 1).permute(1, 0, 2) for x in (cache.kd, cache.vd))
            qs = q[at:at + n].double().permute(1, 0, 2)
            score = (qs @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(score, dim=2)
            p = torch.nan_to_num(torch.exp(score - norm[:, :, None]), nan=0.0)
            out[at:at + n], mag[at:at + n] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
            lse[at:at + n] = norm.t()
            unit = cache.v_scale[cache.table[s].long().clamp(min=0)].double().repeat_interleave(cache.page, 0)[:length].t().repeat_interleave(group, 0)  # [heads, length]
            codes = torch.where(unit[:, :, None] > 0, v.abs() / unit[:, :, None], 0.0)
            most = (p * unit[:, None]).amax(dim=2)
            least[at:at + n] = (2.0 ** -36 * most[:, :, None] * (seen.double() @ codes)).transpose(0, 1)
            if cache.code == "i8":
                least[at:at + n] += 2.0 ** -12 * (p * unit[:, None]).sum(dim=2).t()[:, :, None]
            size = (qs.norm(dim=2)[:, :, None] * k.norm(dim=2)[:, None]).masked_fill(~seen, 0.0)
            spread[at:at + n] = scale * size.amax(dim=2).t()
        at += n
    return (out, lse, mag, spread), least
