"""The operators around an 8-bit cache by their definitions, in 64 bits, and how far a result may be from them."""
import math

import torch

LARGEST = {"i8": 127.0, "e4m3": 448.0}


def code_values(codes, code):
    return codes.view(torch.int8 if code == "i8" else torch.float8_e4m3fn).double()


class Cache:
    """A cache that holds `lengths` tokens a sequence.  Everything that no query may see is filled with what would show: NaN codes
    (E4M3) or the largest ones (int8), table entries that are no pages."""

    def __init__(self, code, lengths, kv_heads, dim, page, seed, token_major=False, spare_pages=2, room=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.code, self.page, self.kv_heads, self.dim = code, page, kv_heads, dim
        wide = max(1, -(-(max(lengths) + room) // page)) + 1
        pages = sum(-(-(n + room) // page) for n in lengths) + spare_pages
        shape = (pages, page, kv_heads, dim) if token_major else (pages, kv_heads, page, dim)
        junk = 0x7F
        self.k, self.v = (torch.full(shape, junk, dtype=torch.uint8, device="cuda") for _ in range(2))
        if token_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.k_scale, self.v_scale = (torch.full((pages, kv_heads), math.nan, device="cuda") for _ in range(2))
        self.table = torch.full((len(lengths), wide), -7, dtype=torch.int32)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.kd, self.vd = [], []  # per sequence, in 64 bits: [length, kv_heads, dim]
        for s, n in enumerate(lengths):
            mine = [order.pop() for _ in range(-(-(n + room) // page))]
            self.table[s, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            for codes, scales, kept, width in ((self.k, self.k_scale, self.kd, 1.0), (self.v, self.v_scale, self.vd, 0.3)):
                x = width * torch.randn((n, kv_heads, dim), generator=g, device="cuda")
                held = torch.zeros((n, kv_heads, dim), dtype=torch.float64, device="cuda")
                for b in range(-(-n // page)):
                    lo, hi = b * page, min(n, (b + 1) * page)
                    scale = x[lo:hi].abs().amax(dim=(0, 2)) / LARGEST[code] * (0.5 + torch.rand(kv_heads, generator=g, device="cuda"))
                    unit = x[lo:hi] / scale[:, None]
                    c = unit.round().clamp(-127, 127).to(torch.int8) if code == "i8" else unit.clamp(-448, 448).to(torch.float8_e4m3fn)
                    codes[mine[b], :, :hi - lo] = c.view(torch.uint8).transpose(0, 1)
                    scales[mine[b]] = scale
                    held[lo:hi] = code_values(c, code) * scale.double()[:, None]
                kept.append(held)
        self.table = self.table.cuda()

    def operands(self, pa):
        return (self.k, self.v, self.k_scale, self.v_scale, self.table, self.lengths, pa.I8 if self.code == "i8" else pa.E4M3)


def starts(counts):
    s = [0]
    for n in counts:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device="cuda")


def attention(q, cache, counts, causal=True, window=0, scale=None):
    """(out, lse, magnitude, spread) in 64 bits: magnitude = sum p |v|, spread = the largest scale |q| |k| of a visible key."""
    tokens, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    spread = torch.zeros((tokens, heads), dtype=torch.float64, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        length = int(cache.lengths[s])
        if n and length:
            group = heads // cache.kv_heads
            k, v = (x[s].repeat_interleave(group, 1).permute(1, 0, 2) for x in (cache.kd, cache.vd))
            qs = q[at:at + n].double().permute(1, 0, 2)
            score = qs @ k.transpose(1, 2) * scale
            place = length - n + torch.arange(n, device="cuda")[:, None]
            key = torch.arange(length, device="cuda")[None]
            seen = torch.ones((n, length), dtype=torch.bool, device="cuda")
            if causal:
                seen &= key <= place
            if window:
                seen &= key > place - window
            score = score.masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(score, dim=2)
            p = torch.nan_to_num(torch.exp(score - norm[:, :, None]), nan=0.0)
            out[at:at + n], mag[at:at + n] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
            lse[at:at + n] = norm.t()
            size = (qs.norm(dim=2)[:, :, None] * k.norm(dim=2)[:, None]).masked_fill(~seen, 0.0)
            spread[at:at + n] = scale * size.amax(dim=2).t()
        at += n
    return out, lse, mag, spread


def check_attention(got, ref, lse=None):
    """Half a unit of the result's type (2^-9 of bf16, 2^-12 of f16; doubled for a result beside a power of two), weights rounded to f16
    (2^-12 each, and as much again for those near the smallest), sums and scores in f32: scores are off by some 2^-20 of |q| |k|, weights by
    as much of themselves."""
    out, norm, mag, spread = ref
    unit = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    score = 2.0 ** -20 * spread + 2.0 ** -20
    tol = unit * out.abs() + (2.0 ** -11 + 2 * score[:, :, None]) * mag + 1e-7 * (mag > 0)
    off = (got.double() - out).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float((off / tol.clamp(min=1e-30)).max()))
    if lse is not None:
        empty = torch.isinf(norm)
        assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
        assert bool(((lse.double() - norm).abs()[~empty] <= (score + 2.0 ** -20 * norm.abs())[~empty] + 2.0 ** -20).all()), \
            float((lse.double() - norm).abs()[~empty].max())
