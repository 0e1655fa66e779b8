"""Attention calls that split the keys of some rows and not of others: single
tokens and few rows in one kernel, chunks in another, each with partial sums of
its own, or none."""
import pytest
import torch

from test_gpu_paged_attention import DT, _cache, _check, _cu

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _cols(kv_lens, page):
    return max((n + page - 1) // page for n in kv_lens)


# Tables much wider than the sequences, which is what the splits go by: chunks beside few
# tokens (sums of the few rows by themselves), many tokens beside a chunk (sums by
# tokens), tokens with offsets, short chunks alone, one long prompt.
CALLS = [([1, 400, 1, 3, 0, 16], [2000, 0, 70, 5, 33, 900]), ([1] * 50 + [40, 1], [37 * i % 700 for i in range(52)]),
         ([1] * 5, [0, 1, 63, 700, 64]), ([7, 2, 15], [600, 0, 90]), ([600], [0]), ([1, 130, 2], [0, 1500, 31])]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,H,D", [(4, 1, 64), (8, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("call", range(len(CALLS)))
def test_wide_tables(att, kind, dtype, heads, H, D, call):
    q_lens, ctx = CALLS[call]
    gen = torch.Generator().manual_seed(call)
    kv_lens = [c + n for c, n in zip(ctx, q_lens)]
    for keys in (8192, 131072):
        cache, table = _cache(att, gen, kv_lens, H, D, 16, kind, keys // 16 - _cols(kv_lens, 16))
        T = sum(q_lens)
        q = (1.5 * torch.randn((T, heads, D), generator=gen)).to(DT[dtype])
        lens = torch.tensor(kv_lens, dtype=torch.int32).cuda()
        # The rows lie in the middle of the call's, whose others stay.
        wide = torch.full((T + 9, heads, D), 7.0, dtype=q.dtype, device="cuda")
        x = torch.zeros_like(wide)
        x[5:5 + T] = q.cuda()
        got = att.paged_attention(x, cache, table.cuda(), lens, (_cu(q_lens) + 5).cuda(), out=wide)
        assert got is wide and (wide[:5] == 7).all() and (wide[5 + T:] == 7).all()
        _check(got[5:5 + T], q, cache, table, kv_lens, q_lens, D ** -0.5, DT[dtype])


def test_a_workspace_that_holds_junk(att):
    """Nothing is read from a workspace that the call did not write."""
    gen = torch.Generator().manual_seed(9)
    for q_lens, ctx in CALLS:
        kv_lens = [c + n for c, n in zip(ctx, q_lens)]
        cache, table = _cache(att, gen, kv_lens, 2, 128, 16, "int8", 600)
        q = torch.randn((sum(q_lens), 8, 128), generator=gen).cuda()
        args = (q, cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), _cu(q_lens).cuda())
        want = att.paged_attention(*args)
        _, n = att._workspace((2, 16, 128, q.shape[0], len(q_lens), 8, 0, table.shape[1], True), "paged", q.device)
        empty = torch.empty
        for junk in (0xFF, 0x00, 0x7F):
            def filled(*a, **kw):
                t = empty(*a, **kw)
                if t.dtype is torch.uint8:
                    t.fill_(junk)
                return t
            torch.empty = filled
            try:
                got = att.paged_attention(*args)
            finally:
                torch.empty = empty
            assert torch.equal(got, want), (n, junk)
