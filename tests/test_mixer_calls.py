"""What the token mixers' host parts make of their arguments, on the CPU: copies
of rows that the kernels cannot load, and the workspaces that calls ask for."""
import pytest
import torch

from breeze_amd import attention as att


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_that_need_a_copy(dtype):
    """One token of rows with an odd stride counts as contiguous whatever its
    address: it is copied too, to where 16-byte loads are aligned."""
    wide = torch.arange(3 * 257, dtype=torch.float32).to(dtype).view(3, 257)
    for t in (wide[:, 1:].view(3, 4, 64), wide[:, 1:].view(3, 4, 64)[:1], wide[:, 1:].view(3, 4, 64)[1:2],
              wide[:1, 1:65].view(1, 1, 64), wide.view(-1)[1:65].view(1, 1, 64), wide[:, ::2][:, :128].view(3, 2, 64)):
        got = att._rows(t, "t")
        st = got.stride()
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0
        assert st[2] == 1 and st[0] % 4 == 0 and st[1] % 4 == 0
    t = torch.zeros((3, 2, 128), dtype=dtype)
    assert att._rows(t, "t") is t
    assert att._rows(t[:, :, :64], "t").data_ptr() == t.data_ptr()  # read in place
