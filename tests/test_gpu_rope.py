"""Rotary positions against their definition in 64 bits."""
import math

import pytest
import torch

from test_gpu_parity import pa  # noqa: F401

pytestmark = pytest.mark.gpu
#: half a unit of a result's type, and of f32 three roundings of products and their sum
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def turned(x, table, positions, interleaved, backward):
    """The result and what its rounding may be off by, in 64 bits."""
    x, rot = x.double(), table.shape[1]
    half = rot // 2
    t = table.double()[positions.long()][:, None]
    cos, sin = t[..., :half], t[..., half:] * (-1 if backward else 1)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :half], x[..., half:rot])
    out, size = x.clone(), torch.zeros_like(x)
    for at, p, q in ((0, a * cos, -b * sin), (1, a * sin, b * cos)):
        to = (Ellipsis, slice(at, rot, 2)) if interleaved else (Ellipsis, slice(at * half, (at + 1) * half))
        out[to], size[to] = p + q, p.abs() + q.abs()
    return out, size


def check(got, x, table, positions, interleaved, backward):
    ref, size = turned(x, table, positions, interleaved, backward)
    unit = UNIT[got.dtype]
    smallest = 2.0 ** -24 if got.dtype == torch.float16 else 0.0  # (f16 has subnormals within reach)
    tol = unit * ref.abs() + 2.0 ** -23 * size + smallest
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() - tol).max())
    assert torch.equal(got[..., table.shape[1]:], x[..., table.shape[1]:])


def inputs(tokens, heads, dim, dtype, seed, rows):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype),
            torch.randint(0, rows, (tokens,), generator=g, device="cuda", dtype=torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 128, 128), (3, 72, 128, 128), (517, 5, 80, 32), (33, 7, 64, 64), (9, 3, 256, 64), (5, 2, 6, 2), (11, 3, 96, 90),
                                                  (2, 3, 7, 4), (70001, 1, 8, 8)])
def test_against_the_definition(pa, dtype, interleaved, tokens, heads, dim, rot):  # noqa: F811
    table = pa.rope_table(3000, rot)
    x, positions = inputs(tokens, heads, dim, dtype, tokens, 3000)
    for backward in (False, True):
        check(pa.rope(x, table, positions, interleaved=interleaved, backward=backward), x, table, positions, interleaved, backward)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_views_and_in_place(pa, interleaved, offset):  # noqa: F811
    """The queries and keys of a fused product; rows that start on any element; the result in place."""
    table = pa.rope_table(500, 64)
    whole, positions = inputs(40, 9, 144, torch.bfloat16, 3, 500)
    x = whole[:, 1:7, offset:offset + 128]
    before = whole.clone()
    expected = pa.rope(x.contiguous(), table, positions, interleaved=interleaved)
    check(expected, x, table, positions, interleaved, False)
    out = torch.zeros((40, 9, 150), dtype=torch.bfloat16, device="cuda")[:, 2:8, 3:131]
    assert torch.equal(pa.rope(x, table, positions, interleaved=interleaved, out=out), expected)
    assert pa.rope(x, table, positions, interleaved=interleaved, out=x) is x
    assert torch.equal(x, expected)
    x.copy_(before[:, 1:7, offset:offset + 128])
    assert torch.equal(whole, before)


def test_positions_outside_the_table(pa):  # noqa: F811
    table = pa.rope_table(100, 32)
    x, _ = inputs(5, 3, 64, torch.float16, 1, 100)
    positions = torch.tensor([0, -1, 99, 100, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out = pa.rope(x, table, positions)
    for t in (1, 3, 4):
        assert bool(out[t, :, :32].isnan().all()) and torch.equal(out[t, :, 32:], x[t, :, 32:])
    check(out[[0, 2]], x[[0, 2]], table, positions[[0, 2]], False, False)
    assert torch.equal(out[0], x[0])  # (position 0 turns nothing)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient(pa, interleaved):  # noqa: F811
    """backward is the gradient of sum(w * rope(x)): by the formula, and by differences along random directions (the map is linear, so a
    difference of any step is the derivative to rounding)."""
    table = pa.rope_table(4096, 48, magnitude=1.25)
    x, positions = inputs(20, 4, 64, torch.float32, 5, 4096)
    w, d = inputs(20, 4, 64, torch.float32, 6, 1)[0], inputs(20, 4, 64, torch.float32, 7, 1)[0]
    grad = pa.rope(w, table, positions, interleaved=interleaved, backward=True)
    check(grad, w, table, positions, interleaved, True)
    change = (pa.rope(x + d, table, positions, interleaved=interleaved).double() - pa.rope(x - d, table, positions, interleaved=interleaved).double()) / 2
    left, right = (w.double() * change).sum(), (grad.double() * d.double()).sum()
    scale = float((w.double().abs() * change.abs()).sum())
    assert abs(float(left - right)) <= 2.0 ** -20 * scale


@pytest.mark.parametrize("kw", [{}, {"base": 500000.0}, {"factor": 4.0}, {"factor": 8.0, "ramp_low": 8.0, "ramp_high": 24.0, "magnitude": 1.2079},
                                {"factor": 32.0, "ramp_low": -3.0, "ramp_high": 7.5}])
def test_the_table(pa, kw):  # noqa: F811
    rows, rot = 131072, 64
    table = pa.rope_table(rows, rot, **kw)
    low, high, factor = kw.get("ramp_low", 0.0), kw.get("ramp_high", 0.0), kw.get("factor", 1.0)
    f = []
    for i in range(rot // 2):
        t = 1.0 if i >= high else 0.0 if i <= low else (i - low) / (high - low)
        g = kw.get("base", 10000.0) ** (-2 * i / rot)
        f.append(g * (1 - t) + g * t / factor)
    at = torch.tensor([0, 1, 2, 1000, 65537, 131071])
    angle = at.double()[:, None] * torch.tensor(f, dtype=torch.float64)
    ref = torch.cat([angle.cos(), angle.sin()], dim=1) * kw.get("magnitude", 1.0)
    got = table[at.cuda()].double().cpu()
    # one rounding to f32; the angle in 64 bits is off by a few 2^-53 of 1.3e5
    assert bool(((got - ref).abs() <= 2.0 ** -24 * ref.abs() + 2e-10).all()), float((got - ref).abs().max())


def test_captured(pa):  # noqa: F811
    table = pa.rope_table(300, 128)
    x, positions = inputs(50, 8, 128, torch.bfloat16, 8, 300)
    pa.rope(x, table, positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.rope(x, table, positions)
    for i in range(3):
        x.mul_(1.5)
        positions.add_(1).remainder_(300)
        graph.replay()
        assert torch.equal(out, pa.rope(x, table, positions)), i
    assert math.isfinite(float(out.float().sum()))
