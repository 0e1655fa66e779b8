"""A row's result does not depend on keys that it does not see, however large
their values are."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
# Rows of 16 a workgroup, of 128, of 128 over an unpacked copy; heads of 256 take the
# second only among many sequences (the last).
@pytest.mark.parametrize("q_lens", [[3], [40], [300], [1] * 60 + [36]])
def test_a_later_tokens_large_values(att, kind, dtype, D, q_lens):
    gen = torch.Generator().manual_seed(1)
    n, ctx, page = q_lens[-1], 21, 16
    T, B, kv = sum(q_lens), len(q_lens), ctx + q_lens[-1]
    P = (kv + page - 1) // page
    cache = att.KVCache.empty(P, page, 1, D, kind)
    k, v = (torch.randn((kv, 1, D), generator=gen).cuda() for _ in range(2))
    at = torch.arange(kv, dtype=torch.int32).cuda()
    att.kv_write(cache, k, v, at)
    q = torch.randn((T, 6, D), generator=gen).to(DT[dtype]).cuda()
    table = torch.arange(P, dtype=torch.int32).expand(B, -1).cuda()
    cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    lens = torch.tensor([ctx] * (B - 1) + [kv], dtype=torch.int32).cuda()
    want = att.paged_attention(q, cache, table, lens, cu)
    for size in (1e4, 1e12, 1e30):
        att.kv_write(cache, k[-1:], v[-1:] * size, at[-1:])
        got = att.paged_attention(q, cache, table, lens, cu)
        assert torch.equal(got[:-1], want[:-1]), size
