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
    tokens, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
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
            size = (qs.norm(dim=2)[:, :, None] * k.norm(dim=2)[:, None]).masked_fill(~seen, 0.0)
            spread[at:at + n] = scale * size.amax(dim=2).t()
        at += n
    return out, lse, mag, spread
