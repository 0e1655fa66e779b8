"""Attention whose scores leave the usual range."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
