"""Attention whose scores leave the usual range: overflow, queries that are no
numbers, softmax scales at the ends of what is accepted."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _setup(att, gen, kv, D, page=16, k_size=1.0, kind="int8"):
    P = (kv + page - 1) // page
    cache = att.KVCache.empty(P, page, 1, D, kind)
    k, v = (torch.randn((kv, 1, D), generator=gen) for _ in range(2))
    att.kv_write(cache, (k_size * k).cuda(), v.cuda(), torch.arange(kv, dtype=torch.int32).cuda())
    return cache, torch.arange(P, dtype=torch.int32)[None].cuda(), v


def _cu(q_lens):
    return torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


# 16 rows a workgroup, split and not; 128 rows, split and not; the same over a copy
# (heads of 256 take it for all of these).
FORMS = [(1, 3000), (1, 20), (40, 3000), (40, 60), (200, 3000), (200, 230)]


@pytest.mark.parametrize("n,kv", FORMS)
@pytest.mark.parametrize("D", [64, 256])
def test_scores_past_fp32(att, n, kv, D):
    """Keys of 1e37 and queries of 1e5: no row has a finite largest score, whether its
    keys are split or not; none is left as the output was."""
    gen = torch.Generator().manual_seed(1)
    cache, table, _ = _setup(att, gen, kv, D, k_size=1e37)
    q = (1e5 * torch.randn((n, 4, D), generator=gen)).cuda()
    out = torch.full_like(q, 7.0)
    att.paged_attention(q, cache, table, torch.tensor([kv], dtype=torch.int32).cuda(), _cu([n]), out=out)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,kv", FORMS)
@pytest.mark.parametrize("D", [64, 256])
def test_queries_of_nan_that_see_nothing(att, dtype, n, kv, D):
    """Zeros, as for any row that sees no key, in one sequence without keys, one with
    fewer keys than rows and one whose pages are not the cache's; NaN where such a
    row sees a key; the other rows as they are."""
    gen = torch.Generator().manual_seed(2)
    cache, table, _ = _setup(att, gen, kv, D)
    n = max(n, 2)
    q = torch.randn((4 * n, 3, D), generator=gen).to(DT[dtype])
    table = table.repeat(4, 1)
    table[2] = -1
    lens = torch.tensor([0, n // 2, kv, kv], dtype=torch.int32).cuda()
    clean = att.paged_attention(q.cuda(), cache, table, lens, _cu([n] * 4))
    bad = torch.zeros((4 * n, 3), dtype=torch.bool)
    bad[::3, 1] = bad[1::3, 0] = True
    x = q.clone()
    x[bad] = float("nan")
    x[0, 0], x[n, 2, 1] = float("inf"), -float("inf")
    bad[0, 0] = bad[n, 2] = True
    got = att.paged_attention(x.cuda(), cache, table, lens, _cu([n] * 4)).cpu()
    sees = torch.ones(4 * n, dtype=torch.bool)
    sees[:n] = sees[2 * n:3 * n] = False
    sees[n:n + n - n // 2] = False
    assert torch.isnan(got[bad & sees[:, None]]).all()
    assert not got[~sees].any() and not torch.isnan(got[~sees]).any()
    assert torch.equal(got[~bad], clean.cpu()[~bad])


@pytest.mark.parametrize("n,kv", FORMS)
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("scale,size", [(1e-30, 1.0), (1e-30, 1e-30), (1e-37, 1e-30)])
def test_softmax_scales_that_leave_no_difference(att, n, kv, D, scale, size):
    """A scale, or a scale and queries, so small that all seen keys weigh alike: the
    mean of the values.  kv sums of fp32 and weights of 22 bits."""
    gen = torch.Generator().manual_seed(3)
    cache, table, _ = _setup(att, gen, kv, D)
    v = att.kv_read(cache, torch.arange(kv, dtype=torch.int32).cuda(), torch.float32)[1].cpu().double()[:, 0]
    q = (size * torch.randn((n, 4, D), generator=gen)).cuda()
    got = att.paged_attention(q, cache, table, torch.tensor([kv], dtype=torch.int32).cuda(), _cu([n]), scale=scale)
    want = (v.cumsum(0) / torch.arange(1, kv + 1).double()[:, None])[kv - n:]
    mean = (v.abs().cumsum(0) / torch.arange(1, kv + 1).double()[:, None])[kv - n:]
    bound = mean * (kv * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -30 * kv * v.abs().max()
    assert ((got.cpu().double() - want[:, None]).abs() <= bound[:, None]).all()


@pytest.mark.parametrize("n,kv", FORMS)
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("scale,size", [(1.0, 1e6), (1.0, 1e8), (1.0, 1e15), (1e20, 1e15)])
def test_scores_so_large_that_one_key_is_left(att, n, kv, D, scale, size):
    """Scores whose differences are all past what the softmax can tell from 0: the
    value of the largest one's key, whatever the scores' own last bits amount to."""
    gen = torch.Generator().manual_seed(4)
    cache, table, _ = _setup(att, gen, kv, D)
    at = torch.arange(kv, dtype=torch.int32).cuda()
    k, v = (t.cpu().double()[:, 0] for t in att.kv_read(cache, at, torch.float32))
    q = size * torch.randn((n, 4, D), generator=gen)
    got = att.paged_attention(q.cuda(), cache, table, torch.tensor([kv], dtype=torch.int32).cuda(), _cu([n]), scale=scale)
    s = torch.einsum("nhd,kd->nhk", q.double(), k)
    s.masked_fill_((torch.arange(kv)[None] > torch.arange(kv - n, kv)[:, None])[:, None], -float("inf"))
    want = v[s.argmax(-1)]
    # The value itself, its weight held in 22 bits and relative to the tile's largest value.
    bound = want.abs() * 2.0 ** -20 + 2.0 ** -30 * kv * v.abs().max()
    two = s.topk(2, dim=-1).values
    clear = (two[..., 0] - two[..., -1]) > 1e-4 * two[..., 0].abs()  # no two keys near enough to swap places
    assert clear.double().mean() > 0.9
    assert ((got.cpu().double() - want).abs() <= bound)[clear].all()
