"""Keys and values quantized into cache pages and read back, against the
64-bit definition: stored numbers and scales are equal, and what is read back
is the product rounded once."""
import pytest
import torch

from mixers_plain import page_values, quantize

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _rows(gen, T, H, D, dtype):
    x = torch.randn((T, H, D), generator=gen) * torch.exp(2 * torch.randn((T, H, 1), generator=gen))
    return x.to(dtype)


def _where(slots, page):
    return (slots.long() // page, slice(None), slots.long() % page)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 64, 16), (1, 4, 256, 16), (77, 3, 128, 32), (515, 2, 64, 128),
                                        (129, 5, 256, 1024)])
def test_written_and_read_back(att, kind, dtype, T, H, D, page):
    gen = torch.Generator().manual_seed(T + H + D)
    k, v = _rows(gen, T, H, D, DT[dtype]), _rows(gen, T, H, D, DT[dtype])
    pages = (T + page - 1) // page + 2
    slots = torch.randperm(pages * page, generator=gen)[:T].to(torch.int32)
    cache = att.KVCache.empty(pages, page, H, D, kind)
    att.kv_write(cache, k.cuda(), v.cuda(), slots.cuda())
    for dt in DT.values():
        got = att.kv_read(cache, slots.cuda(), dt)
        for g, x, ps, sc in ((got[0], k, cache.k, cache.k_scale), (got[1], v, cache.v, cache.v_scale)):
            y, s = quantize(x.double(), kind)
            at = _where(slots, page)
            assert torch.equal(page_values(ps)[at], y)
            assert torch.equal(sc.cpu()[at].double(), s)
            assert torch.equal(g.cpu(), (y.float() * s.float().unsqueeze(-1)).to(dt))
    # Nothing else of the cache was written.
    rest = torch.ones((pages, page), dtype=torch.bool)
    rest[slots.long() // page, slots.long() % page] = False
    for ps, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert not page_values(ps).permute(0, 2, 1, 3)[rest].any()
        assert not sc.cpu().permute(0, 2, 1)[rest].any()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_values_at_borders(att, kind):
    """Halves between two stored numbers, whole rows of one magnitude, zeros,
    tiny, huge and subnormal rows, infinities and NaN."""
    D = 64
    half = torch.arange(D).float() + 0.5
    rows = [torch.cat([half[:-1], torch.tensor([127.0])]), torch.zeros(D), torch.full((D,), -3.0),
            torch.randn(D, generator=torch.Generator().manual_seed(1)) * 1e-38,
            torch.randn(D, generator=torch.Generator().manual_seed(2)) * 1e-42,
            torch.randn(D, generator=torch.Generator().manual_seed(3)) * 3e37,
            torch.full((D,), 1e-45), torch.linspace(-448, 448, D), torch.linspace(-449, 449, D),
            torch.linspace(-1, 1, D) * 2.0 ** -9, torch.full((D,), 2.0 ** -130)]
    nan, inf = torch.randn(D), torch.randn(D)
    nan[5], inf[9] = float("nan"), -float("inf")
    x = torch.stack(rows + [nan, inf]).unsqueeze(1)
    T = x.shape[0]
    cache = att.KVCache.empty(1, 16, 1, D, kind)
    slots = torch.arange(T, dtype=torch.int32).cuda()
    att.kv_write(cache, x.cuda(), x.flip(0).contiguous().cuda(), slots)
    for ps, sc, src in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, x.flip(0))):
        y, s = quantize(src.double(), kind)
        assert torch.equal(page_values(ps)[0, 0, :T], y[:, 0])
        assert torch.equal(sc.cpu()[0, 0, :T].double().nan_to_num(-1), s[:, 0].nan_to_num(-1))
    back = att.kv_read(cache, slots, torch.float32)[0].cpu()
    assert torch.isnan(back[T - 2:]).all() and torch.isfinite(back[:T - 2]).all()


def test_slots_outside_the_cache(att):
    gen = torch.Generator().manual_seed(3)
    x = _rows(gen, 6, 2, 64, torch.float32).cuda()
    cache = att.KVCache.empty(2, 16, 2, 64)
    slots = torch.tensor([-1, 3, 32, -2147483648, 31, 2147483647], dtype=torch.int32).cuda()
    att.kv_write(cache, x, x, slots)
    k, v = att.kv_read(cache, slots, torch.float32)
    assert not k[[0, 2, 3, 5]].any() and not v[[0, 2, 3, 5]].any()
    assert k[[1, 4]].abs().sum() > 0
    assert int((cache.k_scale != 0).sum()) == 4


@pytest.mark.parametrize("dtype", list(DT))
def test_views_of_a_wider_projection(att, dtype):
    """k and v as columns of one buffer, and rows that need a copy first."""
    gen = torch.Generator().manual_seed(4)
    H, D, T = 4, 128, 37
    for width, lead in ((3 * H * D, 0), (3 * H * D + 4, 4), (2 * H * D + 3, 1)):
        buf = torch.randn((T, width), generator=gen).to(DT[dtype]).cuda()
        k = buf[:, lead:lead + H * D].view(T, H, D)
        v = buf[:, lead + H * D:lead + 2 * H * D].view(T, H, D)
        slots = torch.randperm(64, generator=gen)[:T].to(torch.int32).cuda()
        a, b = att.KVCache.empty(4, 16, H, D), att.KVCache.empty(4, 16, H, D)
        att.kv_write(a, k, v, slots)
        att.kv_write(b, k.clone(), v.clone(), slots)
        for f in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(a, f), getattr(b, f))


def test_far_pages(att):
    """Rows of the cache past 2^31 bytes."""
    P, page, H, D = 2100, 1024, 4, 256
    cache = att.KVCache(*(torch.empty((P, H, page, D), dtype=torch.int8, device="cuda") for _ in range(2)),
                        *(torch.empty((P, H, page), dtype=torch.float32, device="cuda") for _ in range(2)))
    gen = torch.Generator().manual_seed(5)
    x = _rows(gen, 3, H, D, torch.float32)
    slots = torch.tensor([0, P * page - 1, P * page - 1024], dtype=torch.int32)
    att.kv_write(cache, x.cuda(), (2 * x).cuda(), slots.cuda())
    k, v = att.kv_read(cache, slots.cuda(), torch.float32)
    y, s = quantize(x.double(), "int8")
    assert torch.equal(k.cpu(), y.float() * s.float().unsqueeze(-1))
    assert torch.equal(v.cpu(), 2 * k.cpu())


def test_captured_write_and_read(att):
    gen = torch.Generator().manual_seed(6)
    xs = [_rows(gen, 9, 2, 128, torch.bfloat16).cuda() for _ in range(4)]
    slots = torch.arange(9, dtype=torch.int32).cuda()
    cache, plain = att.KVCache.empty(1, 16, 2, 128, "fp8"), att.KVCache.empty(1, 16, 2, 128, "fp8")
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        att.kv_write(cache, x, x, slots)
        k, v = att.kv_read(cache, slots, torch.float32)
    for y in xs:
        x.copy_(y)
        graph.replay()
        att.kv_write(plain, y, y, slots)  # eager work between the replays
        want = att.kv_read(plain, slots, torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
