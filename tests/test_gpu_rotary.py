"""Rotary positions against their 64-bit form: layouts, parts of the head,
scalings, far positions, views, outputs in place, a captured graph."""
import math

import pytest
import torch

from mixers_plain import half_step

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _turn(x, positions, freqs, layout, amplitude):
    """(y, bound) in fp64 on the CPU; freqs in radians a position."""
    x = x.cpu().double()
    r, half = 2 * len(freqs), len(freqs)
    angle = positions.cpu().double()[:, None, None] * torch.tensor(freqs, dtype=torch.float64)
    c, s = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
    at = torch.arange(half)
    i, j = (at, at + half) if layout == "half" else (2 * at, 2 * at + 1)
    y, bound = x.clone(), torch.zeros_like(x)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    # Sine and cosine: four last places, an angle within 2^-25 of a quarter turn, the
    # amplitude's rounding; then two products and their sum.
    size = (a.abs() + b.abs()) * amplitude * (4 + 1 + 1 + 2) * 2.0 ** -24
    bound[..., i], bound[..., j] = size, size
    return y, bound


def _check(got, x, positions, freqs, layout, amplitude):
    y, bound = _turn(x, positions, freqs, layout, amplitude)
    tiny = torch.finfo(got.dtype).smallest_normal
    # Values that are copied stay as they are.
    turned = torch.zeros(x.shape[-1], dtype=torch.bool)
    turned[:2 * len(freqs)] = True
    assert torch.equal(got.cpu()[..., ~turned], x.cpu()[..., ~turned])
    off = (got.cpu().double() - y).abs()[..., turned]
    allowed = (bound + half_step(got.dtype) * (y.abs() + bound).clamp_min(tiny))[..., turned]
    assert (off <= allowed).all(), (off / allowed.clamp_min(1e-300)).max().item()


def _freqs(dim, base=10000.0):
    return [base ** (-2 * i / dim) for i in range(dim // 2)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D,rot", [(256, 64), (128, 128), (64, 50), (64, 8), (80, 24), (128, 2), (6, 4), (96, 48)])
@pytest.mark.parametrize("T,heads,kv_heads", [(1, 24, 4), (3, 1, 1), (77, 5, 2)])
def test_layouts(att, layout, dtype, D, rot, T, heads, kv_heads):
    gen = torch.Generator().manual_seed(T * D + rot)
    wide = torch.randn((T, (heads + kv_heads) * D + 16), generator=gen).to(DT[dtype]).cuda()
    q, k = wide[:, :heads * D].view(T, heads, D), wide[:, heads * D:(heads + kv_heads) * D].view(T, kv_heads, D)
    positions = torch.randint(0, 200000, (T,), generator=gen, dtype=torch.int32).cuda()
    rope = att.Rotary(rot, layout=layout)
    before = wide.clone()
    qo, ko = att.rotary(rope, q, k, positions)
    assert torch.equal(wide, before)
    for got, x in ((qo, q), (ko, k)):
        _check(got, x, positions, _freqs(rot), layout, 1.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_tokens(att, dtype):
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn((2500, h, 128), generator=gen).to(DT[dtype]).cuda() for h in (8, 2))
    positions = (torch.arange(2500, dtype=torch.int32) + 100000).cuda()
    qo, ko = att.rotary(att.Rotary(96, base=1e6, layout="interleaved"), q, k, positions)
    for got, x in ((qo, q), (ko, k)):
        _check(got, x, positions, _freqs(96, 1e6), "interleaved", 1.0)


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_alignment(att, dtype, offset):
    """Rows at every alignment that the type allows, in and out."""
    gen = torch.Generator().manual_seed(offset)
    x = torch.randn((9, 3 * 64 + offset), generator=gen).to(DT[dtype]).cuda()[:, offset:].view(9, 3, 64)
    out = torch.zeros((9, 3, 64 + offset), dtype=DT[dtype], device="cuda")[..., offset:]
    positions = torch.arange(9, dtype=torch.int32).cuda()
    got, none = att.rotary(att.Rotary(64), x, None, positions, (out, None))
    assert got is out and none is None
    _check(out, x, positions, _freqs(64), "half", 1.0)


def test_far_and_negative_positions(att):
    x = torch.ones((6, 1, 64), device="cuda")
    positions = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7], dtype=torch.int32).cuda()
    got, _ = att.rotary(att.Rotary(64), x, None, positions)
    # fp64 angles are 2^31 * 2^-53 off: 2^-22 of a radian.
    y, bound = _turn(x, positions, _freqs(64), "half", 1.0)
    assert ((got.cpu().double() - y).abs() <= bound + 2.0 ** -21 + 2.0 ** -24 * y.abs()).all()
    assert torch.equal(got[0], x[0])


def test_scalings(att):
    dim, factor, original = 64, 8.0, 4096
    x = torch.randn((4, 2, 64), generator=torch.Generator().manual_seed(0)).cuda()
    positions = torch.tensor([1, 500, 4096, 30000], dtype=torch.int32).cuda()
    f = _freqs(dim)
    parts = []
    for w in f:
        keep = min(max((original * w / (2 * math.pi) - 1) / 31, 0), 1)
        parts.append(keep * w + (1 - keep) * w / factor)
    assert parts[0] == f[0] and parts[-1] == f[-1] / factor  # one kept, one divided
    base = [(10000 * factor ** (64 / 62)) ** (-2 * i / dim) for i in range(32)]
    assert abs(base[-1] * factor / f[-1] - 1) < 1e-12
    for rope, freqs, amplitude in (
            (att.Rotary(dim, scaling="linear", factor=factor), [w / factor for w in f], 1.0),
            (att.Rotary(dim, scaling="base", factor=factor), base, 1.0),
            (att.Rotary(dim, scaling="parts", factor=factor, original=original), parts, 0.1 * math.log(factor) + 1),
            (att.Rotary(dim, scaling="parts", factor=factor, original=original, amplitude=1.0), parts, 1.0),
            (att.Rotary(dim, freqs=parts, amplitude=0.5), parts, 0.5)):
        got, _ = att.rotary(rope, x, None, positions)
        _check(got, x, positions, freqs, "half", amplitude)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place(att, layout):
    """In place in a fused projection: only the turned values are written."""
    gen = torch.Generator().manual_seed(3)
    rope = att.Rotary(32, layout=layout)
    wide = torch.randn((700, 3 * 64), generator=gen).cuda()
    before, positions = wide.clone(), torch.arange(700, dtype=torch.int32).cuda()
    q, k = wide[:, :128].view(700, 2, 64), wide[:, 128:].view(700, 1, 64)
    want = att.rotary(rope, before[:, :128].view(700, 2, 64), before[:, 128:].view(700, 1, 64), positions)
    got = att.rotary(rope, q, k, positions, (q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    # One in place, the other apart.
    wide.copy_(before)
    out = torch.empty_like(want[1])
    att.rotary(rope, q, k, positions, (q, out))
    assert torch.equal(q, want[0]) and torch.equal(out, want[1]) and torch.equal(wide[:, 128:], before[:, 128:])


def test_nothing_and_special_values(att):
    rope = att.Rotary(64)
    q = torch.zeros((0, 4, 64), device="cuda")
    got, none = att.rotary(rope, q, None, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 4, 64) and none is None
    x = torch.zeros((2, 1, 64), device="cuda")
    x[0, 0, 3], x[1, 0, 40] = float("nan"), float("inf")
    got, _ = att.rotary(rope, x, None, torch.tensor([5, 5], dtype=torch.int32, device="cuda"))
    bad = ~torch.isfinite(got)
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 35] and bad[1, 0].nonzero().flatten().tolist() == [8, 40]


def test_graph_and_stream(att):
    gen = torch.Generator().manual_seed(8)
    rope = att.Rotary(64)
    q, k = (torch.randn((5, h, 128), generator=gen).cuda() for h in (6, 2))
    positions = torch.arange(5, dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    stream, held = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        got = att.rotary(rope, q, k, positions)
    for step in range(3):
        q.copy_(torch.randn((5, 6, 128), generator=gen))
        positions.add_(1000 * step)
        want = att.rotary(rope, q, k, positions)
        held.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
