"""Attention over the paged cache against a 64-bit form of it, within the
error that its products' documented precision gives each element."""
import pytest
import torch

from mixers_plain import attend, half_step

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _cache(att, gen, kv_lens, H, D, page, kind, extra=0, spread=1.0):
    """A cache whose used rows hold data and whose other rows hold what must not
    matter (NaN scales, e4m3 NaN bytes); table entries past the need are bad."""
    need = [(n + page - 1) // page for n in kv_lens]
    P, cols = sum(need) + 2, max(need + [0]) + extra
    cols = max(cols, 1)
    order = torch.randperm(P, generator=gen).to(torch.int32)
    junk = torch.full((P, H, page, D), 0x7F, dtype=torch.int8)
    pages = [(junk if kind == "int8" else junk.view(torch.float8_e4m3fn)).cuda() for _ in range(2)]
    pages = [p.clone() for p in pages]
    scales = [torch.full((P, H, page), float("nan"), device="cuda") for _ in range(2)]
    cache = att.KVCache(*pages, *scales)
    table = torch.full((len(kv_lens), cols), 1 << 30, dtype=torch.int32)
    at = 0
    for b, (n, c) in enumerate(zip(kv_lens, need)):
        table[b, :c] = order[at:at + c]
        at += c
        if n:
            j = torch.arange(n)
            slots = (table[b].long()[j // page] * page + j % page).to(torch.int32).cuda()
            k = torch.randn((n, H, D), generator=gen) * torch.exp(0.3 * spread * torch.randn((n, H, 1), generator=gen))
            v = torch.randn((n, H, D), generator=gen) * torch.exp(spread * torch.randn((n, H, 1), generator=gen))
            att.kv_write(cache, k.cuda(), v.cuda(), slots)
    return cache, table


def _cu(q_lens):
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def _check(got, q, cache, table, kv_lens, q_lens, scale, dtype, fine=False):
    T = sum(q_lens)
    want, bound = attend(q[:T], cache, table, kv_lens, q_lens, scale, fine or dtype is torch.float32)
    # One rounding to the type: half a step of the value, or of the smallest normal
    # number, below which the steps stay as wide (fp16: 2^-24, so half is 2^-25).
    bound = bound + half_step(dtype) * (want.abs() + bound).clamp_min(torch.finfo(dtype).smallest_normal)
    got = got[:T].cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any()
    is_number = ~torch.isnan(want)
    off, bound = (got - want).abs()[is_number], bound[is_number]
    assert torch.isfinite(bound).all()
    worst = (off / bound).max().item() if off.numel() else 0.0
    print(f"error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0


def _run(att, seed, kind, dtype, heads, H, D, page, q_lens, ctx, extra=0, single=False, scale=None, spread=1.0,
         fine=False):
    gen = torch.Generator().manual_seed(seed)
    kv_lens = [c + n for c, n in zip(ctx, q_lens)]
    cache, table = _cache(att, gen, kv_lens, H, D, page, kind, extra, spread)
    q = (1.5 * torch.randn((sum(q_lens), heads, D), generator=gen)).to(DT[dtype])
    lens = torch.tensor(kv_lens, dtype=torch.int32)
    got = att.paged_attention(q.cuda(), cache, table.cuda(), lens.cuda(), None if single else _cu(q_lens).cuda(),
                              scale)
    _check(got, q, cache, table, kv_lens, q_lens, scale or D ** -0.5, DT[dtype], fine)


ONE = [0, 1, 15, 16, 31, 32, 99, 127, 128, 500]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,H,D,page", [(6, 1, 256, 16), (8, 2, 128, 32), (3, 3, 64, 64), (16, 1, 64, 16),
                                            (48, 2, 128, 16)])
def test_single_tokens(att, kind, dtype, heads, H, D, page):
    _run(att, 1, kind, dtype, heads, H, D, page, [1] * len(ONE), ONE, single=True)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,H,D,page,extra", [(6, 1, 256, 16, 100), (4, 4, 128, 64, 40), (16, 2, 64, 128, 0)])
def test_single_tokens_of_long_contexts(att, kind, dtype, heads, H, D, page, extra):
    """Split over the keys and joined; the table has room for more."""
    _run(att, 2, kind, dtype, heads, H, D, page, [1, 1], [2500, 700], extra, single=True)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,H,D,page", [(6, 1, 256, 16), (8, 2, 128, 32), (3, 3, 64, 64), (130, 1, 64, 16)])
def test_chunks(att, kind, dtype, heads, H, D, page):
    q_lens = [1, 0, 33, 2, 5, 130, 1, 3]
    ctx = [17, 40, 0, 63, 0, 200, 0, 500]
    _run(att, 3, kind, dtype, heads, H, D, page, q_lens, ctx)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("heads,H,D", [(6, 1, 256), (4, 1, 128), (2, 2, 64)])
def test_a_chunk_of_a_long_context(att, dtype, heads, H, D):
    _run(att, 4, "int8", dtype, heads, H, D, 64, [70], [3000], extra=20)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,H,D,page", [(6, 1, 256, 16), (8, 2, 128, 64), (12, 3, 64, 32)])
@pytest.mark.parametrize("q_lens,ctx,extra", [([300], [0], 0), ([1, 260, 2, 400], [300, 77, 0, 63], 3),
                                              ([129], [1500], 9)])
def test_long_chunks(att, kind, dtype, heads, H, D, page, q_lens, ctx, extra):
    """Enough rows a sequence that its keys are unpacked once for all of them."""
    if D == 256 and len(q_lens) == 1 and q_lens[0] == 300 and dtype == "bf16":
        _run(att, 40, kind, dtype, heads, H, D, page, [1300], [5], spread=4.0)
    _run(att, 41, kind, dtype, heads, H, D, page, q_lens, ctx, extra)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,H,D", [(6, 1, 256), (8, 2, 128), (12, 3, 64)])
def test_long_chunks_among_many_sequences(att, kind, dtype, heads, H, D):
    """Copies for the long chunks only, beside single tokens and short chunks."""
    q_lens = [1, 3, 1, 130, 1, 1, 20, 0, 1, 1, 75, 64, 1, 1, 1, 1, 1, 90] + [1] * 12
    ctx = [7 * i % 131 for i in range(len(q_lens))]
    _run(att, 42, kind, dtype, heads, H, D, 16, q_lens, ctx)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("heads,H,D", [(6, 1, 256), (8, 2, 128), (12, 3, 64)])
@pytest.mark.parametrize("q_lens,ctx,extra", [([1, 1, 1], [0, 3, 2000], 0), ([2, 9, 4], [700, 0, 33], 0),
                                              ([20, 33, 1], [7, 0, 60], 0), ([300], [0], 0), ([130, 380], [300, 0], 3)])
def test_fp16_rows_that_take_two_terms(att, kind, heads, H, D, q_lens, ctx, extra):
    """Few rows, or fewer than 512 keys: the output's rounding is the only one to 11 bits."""
    _run(att, 44, kind, "fp16", heads, H, D, 16, q_lens, ctx, extra, single=max(q_lens) == 1, fine=True)


@pytest.mark.parametrize("heads", [17, 128, 129, 300])
def test_many_heads_of_one_key_head(att, heads):
    _run(att, 5, "int8", "bf16", heads, 1, 64, 16, [1, 1], [40, 3], single=True)


def test_scale_and_unlike_values(att):
    """A given softmax scale, and value scales over many powers of two."""
    for dtype in DT:
        _run(att, 6, "int8", dtype, 4, 2, 128, 16, [3, 40], [90, 500], scale=0.5, spread=4.0)
        _run(att, 7, "fp8", dtype, 4, 2, 128, 16, [1, 1], [90, 700], scale=0.02, spread=4.0, single=True)


@pytest.mark.parametrize("dtype", list(DT))
def test_queries_of_any_size(att, dtype):
    """Rows of zeros, tiny and large rows: the scores decide, not the fp16 range."""
    gen = torch.Generator().manual_seed(8)
    for n in (1, 40):
        cache, table = _cache(att, gen, [300], 2, 64, 16, "int8")
        q = torch.randn((n, 4, 64), generator=gen)
        q[0, 0] = 0
        q[0, 1] *= 1e-30 if dtype != "fp16" else 1e-5
        q[0, 2] *= 30
        q[0, 3, 1:] *= 1e-4
        q = q.to(DT[dtype])
        got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor([300], dtype=torch.int32).cuda(),
                                  _cu([n]).cuda())
        _check(got, q, cache, table, [300], [n], 64 ** -0.5, DT[dtype])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("n", [1, 20, 150])
def test_rows_that_see_nothing(att, kind, n):
    """No keys, fewer keys than new tokens, and pages that are not the cache's."""
    gen = torch.Generator().manual_seed(9)
    kv_lens = [0, n // 2, 70, 200, 33]
    cache, table = _cache(att, gen, kv_lens, 2, 128, 16, kind)
    P = cache.num_pages
    table[2] = -1
    table[3, 0], table[3, 3], table[3, 12] = -5, P, 2147483647
    q_lens = [n] * 5
    q = torch.randn((5 * n, 8, 128), generator=gen)
    got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(),
                              _cu(q_lens).cuda())
    _check(got, q, cache, table, kv_lens, q_lens, 128 ** -0.5, torch.float32)
    assert not got[:n].any() and not got[2 * n:3 * n].any()
    # Lengths past the table and negative ones.
    lens = torch.tensor([-3, 1 << 30, -(1 << 31), 2147483647, 33], dtype=torch.int32)
    got = att.paged_attention(q.cuda(), cache, table.cuda(), lens.cuda(), _cu(q_lens).cuda())
    if kind == "fp8":
        # Keys that were never written count as there now, and e4m3 pages may not hold
        # NaN there (kv_write stores none): only the other sequences have values.
        for b in (0, 2, 4):
            part = slice(b * n, b * n + n)
            _check(got[part], q[part], cache, table[b:b + 1], lens[b:b + 1].tolist(), [n], 128 ** -0.5, torch.float32)
        return
    _check(got, q, cache, table, lens.tolist(), q_lens, 128 ** -0.5, torch.float32)


@pytest.mark.parametrize("heads,H", [(4, 1), (34, 1)])
def test_rows_outside_the_sequences_stay(att, heads, H):
    gen = torch.Generator().manual_seed(10)
    for ctx in (40, 3000):
        q_lens = [1, 9]
        cache, table = _cache(att, gen, [ctx + 1, ctx + 9], H, 64, 16, "int8")
        q = torch.randn((17, heads, 64), generator=gen).cuda()
        cu = (_cu(q_lens) + 3).cuda()
        out = torch.full_like(q, 7.0)
        lens = torch.tensor([ctx + 1, ctx + 9], dtype=torch.int32).cuda()
        att.paged_attention(q, cache, table.cuda(), lens, cu, out=out)
        assert (out[:3] == 7).all() and (out[13:] == 7).all()
        _check(out[3:13], q[3:13], cache, table, [ctx + 1, ctx + 9], q_lens, 0.125, torch.float32)
        # Offsets that are no offsets: no fault, and rows outside 0 .. T untouched.
        bad = torch.tensor([-5, 1 << 30, 2], dtype=torch.int32).cuda()
        att.paged_attention(q, cache, table.cuda(), lens, bad)
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [40, 200])
def test_nan_rows_stay_apart(att, n):
    """A query with NaN or infinity spoils its own row; a key that a row does
    not see spoils nothing."""
    gen = torch.Generator().manual_seed(11)
    heads = 4
    cache, table = _cache(att, gen, [100 if n < 100 else n], 1, 64, 16, "int8")
    q = torch.randn((n, heads, 64), generator=gen)
    kv = 100 if n < 100 else n
    lens, cu = torch.tensor([kv], dtype=torch.int32).cuda(), _cu([n]).cuda()
    clean = att.paged_attention(q.cuda(), cache, table.cuda(), lens, cu)
    x = q.clone()
    x[5, 1, 3], x[30, 2, 0] = float("nan"), float("inf")
    got = att.paged_attention(x.cuda(), cache, table.cuda(), lens, cu)
    keep = torch.ones((n, heads), dtype=torch.bool)
    keep[5, 1] = keep[30, 2] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
    assert torch.isnan(got[5, 1]).all() and torch.isnan(got[30, 2]).all()
    # The last key's row turns to NaN: only the last token sees it.
    slot = int(table[0, (kv - 1) // 16]) * 16 + (kv - 1) % 16
    bad = torch.full((1, 1, 64), float("nan")).cuda()
    att.kv_write(cache, bad, bad, torch.tensor([slot], dtype=torch.int32).cuda())
    got = att.paged_attention(q.cuda(), cache, table.cuda(), lens, cu)
    assert torch.equal(got[:-1], clean[:-1]) and torch.isnan(got[-1]).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", [1, 30])
def test_strides_and_outputs(att, dtype, n):
    """Queries as a part of each head's columns, rows that need a copy, a given
    output with its own strides, and the queries themselves as output."""
    gen = torch.Generator().manual_seed(12)
    heads, H, D = 6, 1, 128
    cache, table = _cache(att, gen, [n + 50, n + 800], H, D, 32, "int8")
    lens, cu = torch.tensor([n + 50, n + 800], dtype=torch.int32).cuda(), _cu([n, n]).cuda()
    table = table.cuda()
    wide = torch.randn((2 * n, heads, 2 * D), generator=gen).to(DT[dtype]).cuda()
    q = wide[:, :, :D]
    want = att.paged_attention(q.clone(), cache, table, lens, cu)
    assert torch.equal(att.paged_attention(q, cache, table, lens, cu), want)
    odd = torch.empty((2 * n, heads * D + 1), dtype=q.dtype, device="cuda")[:, 1:].view(2 * n, heads, D)
    odd.copy_(q)
    assert torch.equal(att.paged_attention(odd, cache, table, lens, cu), want)
    out = torch.full((2 * n, heads, 3 * D), 5.0, dtype=q.dtype, device="cuda")
    att.paged_attention(q, cache, table, lens, cu, out=out[:, :, D:2 * D])
    assert torch.equal(out[:, :, D:2 * D], want) and (out[:, :, :D] == 5).all() and (out[:, :, 2 * D:] == 5).all()
    same = q.clone()
    assert att.paged_attention(same, cache, table, lens, cu, out=same) is same
    assert torch.equal(same, want)
    # A table whose rows are a part of a wider one.
    t2 = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    t2[:, 2:-3] = table
    assert torch.equal(att.paged_attention(q, cache, t2[:, 2:-3], lens, cu), want)


def test_repeats_bit_for_bit_on_streams_and_in_graphs(att):
    gen = torch.Generator().manual_seed(13)
    kv = [1500, 40, 700]
    cache, table = _cache(att, gen, kv, 2, 128, 16, "int8")
    table, lens = table.cuda(), torch.tensor(kv, dtype=torch.int32).cuda()
    for q_lens in ([1, 1, 1], [30, 1, 5], [300, 30, 200]):
        cu = None if max(q_lens) == 1 else _cu(q_lens).cuda()
        qs = [torch.randn((sum(q_lens), 8, 128), generator=gen).cuda() for _ in range(4)]
        want = [att.paged_attention(q, cache, table, lens, cu) for q in qs]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got.append(att.paged_attention(q, cache, table, lens, cu))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # Two graphs captured on one stream, replayed on two.
        xs, outs, graphs = [qs[0].clone(), qs[1].clone()], [], []
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                outs.append(att.paged_attention(x, cache, table, lens, cu))
            graphs.append(g)
        for i in range(4):
            xs[0].copy_(qs[i])
            xs[1].copy_(qs[3 - i])
            torch.cuda.synchronize()
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            again = att.paged_attention(qs[i], cache, table, lens, cu)  # eager work between
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[3 - i]) and torch.equal(again, want[i])


def test_far_pages(att):
    """Keys whose cache rows lie past 2^31 bytes."""
    P, page, H, D = 2100, 1024, 4, 256
    cache = att.KVCache(*(torch.zeros((P, H, page, D), dtype=torch.int8, device="cuda") for _ in range(2)),
                        *(torch.zeros((P, H, page), dtype=torch.float32, device="cuda") for _ in range(2)))
    gen = torch.Generator().manual_seed(14)
    small = att.KVCache.empty(2, page, H, D)
    k, v = (torch.randn((1100, H, D), generator=gen).cuda() for _ in range(2))
    j = torch.arange(1100)
    for c, pages in ((cache, [P - 1, 17]), (small, [0, 1])):
        slots = (torch.tensor(pages)[j // page] * page + j % page).to(torch.int32).cuda()
        att.kv_write(c, k, v, slots)
    for n in (1, 50, 600):
        q = torch.randn((n, 8, D), generator=gen).cuda()
        lens, cu = torch.tensor([1100], dtype=torch.int32).cuda(), _cu([n]).cuda()
        a = att.paged_attention(q, cache, torch.tensor([[P - 1, 17]], dtype=torch.int32).cuda(), lens, cu)
        b = att.paged_attention(q, small, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), lens, cu)
        assert torch.equal(a, b)
