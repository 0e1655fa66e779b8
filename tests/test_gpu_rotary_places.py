"""Rotary positions in place in a projection whose heads each hold q, k and v."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 700])
def test_heads_that_hold_all_three(gpu, T, dtype):
    from breeze_amd import attention as att
    gen = torch.Generator().manual_seed(T)
    x = torch.randn((T, 4, 3, 64), generator=gen).to(dtype).cuda()
    rope, positions, before = att.Rotary(32), torch.arange(T, dtype=torch.int32).cuda() + 9, x.clone()
    want = att.rotary(rope, before[:, :, 0].contiguous(), before[:, :, 1].contiguous(), positions)
    q, k = x[:, :, 0], x[:, :, 1]
    got = att.rotary(rope, q, k, positions, (q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(x[:, :, 2], before[:, :, 2])
    with pytest.raises(ValueError, match="lie on one another"):
        att.rotary(rope, q, k, positions, (q, q))
