"""Heads of 256 where the calls have too few rows for a copy of every sequence:
the kernel that unpacks tiles on the way, and copies for the long chunks only;
and what calls with bad offsets leave alone."""
import pytest
import torch

from test_gpu_paged_attention import DT, _cache, _check, _cu

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _copies(hb, q_lens, kv_lens_cols, heads, H, D, page, dtype):
    """Copies of sequences that the call's workspace has room for."""
    one = H * -(-kv_lens_cols * page // 64) * (64 * D * 4 + 1024)
    n = hb._lib.i4_paged_attention_workspace(H, page, D, sum(q_lens), len(q_lens), heads, dtype, kv_lens_cols, 1)
    assert n >= 0
    return n // one


# Rows (tokens times 6): single tokens, then on both sides of 128 (16 rows a
# workgroup up to there) and of 256 (a copy from there on).
MANY = [1] * 20 + [21, 0, 22, 1, 25, 42, 43, 3, 64] + [1] * 35


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
def test_short_and_long_chunks_among_single_tokens(att, hb, kind, dtype):
    heads, H, D, page = 6, 1, 256, 16
    ctx = [11 * i % 157 for i in range(len(MANY))]
    ctx[24], ctx[28] = 700, 1100
    gen = torch.Generator().manual_seed(1)
    kv_lens = [c + n for c, n in zip(ctx, MANY)]
    cache, table = _cache(att, gen, kv_lens, H, D, page, kind)
    # Fewer than 64 rows a sequence: no copy for each, but one for every 256 rows and one more.
    rows = sum(MANY) * 6
    assert 64 <= rows < 64 * len(MANY)
    assert rows // 256 + 1 <= _copies(hb, MANY, table.shape[1], heads, H, D, page, list(DT).index(dtype)) < len(MANY)
    q = (1.5 * torch.randn((sum(MANY), heads, D), generator=gen)).to(DT[dtype])
    got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), _cu(MANY).cuda())
    _check(got, q, cache, table, kv_lens, MANY, D ** -0.5, DT[dtype])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_chunks_of_heads_that_share_nothing(att, hb, kind, dtype):
    """As many key heads as query heads: few rows a sequence, tokens in hundreds."""
    q_lens = [200, 1, 140] + [1] * 30
    ctx = [300, 5, 0] + [3 * i for i in range(30)]
    gen = torch.Generator().manual_seed(2)
    kv_lens = [c + n for c, n in zip(ctx, q_lens)]
    cache, table = _cache(att, gen, kv_lens, 2, 256, 32, kind)
    assert _copies(hb, q_lens, table.shape[1], 2, 2, 256, 32, list(DT).index(dtype)) < len(q_lens)
    q = torch.randn((sum(q_lens), 2, 256), generator=gen).to(DT[dtype])
    got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), _cu(q_lens).cuda())
    _check(got, q, cache, table, kv_lens, q_lens, 1 / 16, DT[dtype])


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("T", [17, 300])
@pytest.mark.parametrize("ctx", [40, 3000])
def test_bad_offsets_write_nothing_past_the_rows(att, D, T, ctx):
    """Offsets that are no offsets: only rows of the given output are written."""
    gen = torch.Generator().manual_seed(3)
    cache, table = _cache(att, gen, [ctx, ctx], 1, D, 16, "int8")
    q = torch.randn((T, 4, D), generator=gen).cuda()
    lens = torch.tensor([ctx, ctx], dtype=torch.int32).cuda()
    wide = torch.full((T + 64, 4, D), 7.0, device="cuda")
    for bad in ([-5, 1 << 30, 2], [T, 0, T], [T + 3, -1, 1 << 30], [-(1 << 31), 2147483647, -1], [5, 5, 5]):
        wide.fill_(7.0)
        att.paged_attention(q, cache, table.cuda(), lens, torch.tensor(bad, dtype=torch.int32).cuda(),
                            out=wide[32:32 + T])
        assert (wide[:32] == 7).all() and (wide[32 + T:] == 7).all()
    assert (wide == 7).all()  # the last offsets hold no row at all


@pytest.mark.parametrize("T", [12, 160])
def test_bad_offsets_of_linear_attention_write_nothing_past_the_rows(att, T):
    gen = torch.Generator().manual_seed(4)
    Hv, Dk, Dv = 2, 64, 48
    q, k = (torch.randn((T, 1, Dk), generator=gen).cuda() / 8 for _ in range(2))
    v, g = torch.randn((T, Hv, Dv), generator=gen).cuda(), -torch.rand((T, Hv), generator=gen).cuda()
    for bad in ([1 << 30, -7, 90, 2], [T, 0, T, 0], [-(1 << 31), 2147483647, -1, 3], [T + 1, T + 2, 1 << 30, -1],
                [4, 4, 4, 4]):
        B = len(bad) - 1
        wide = torch.full((T + 64, Hv, Dv), 9.0, device="cuda")
        states = torch.full((B + 2, Hv, Dk, Dv), 5.0, device="cuda")
        old = torch.randn((B, Hv, Dk, Dv), generator=gen).cuda()
        att.gated_linear_attention(q, k, v, g, g.abs(), old, torch.tensor(bad, dtype=torch.int32).cuda(),
                                   out=wide[32:32 + T], state_out=states[1:-1])
        assert (wide[:32] == 9).all() and (wide[32 + T:] == 9).all()
        assert (states[0] == 5).all() and (states[-1] == 5).all()
    assert (wide == 9).all() and torch.equal(states[1:-1], old)  # no token: the states as they were
