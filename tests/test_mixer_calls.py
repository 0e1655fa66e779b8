"""What the token mixers' host parts make of their arguments, on the CPU: copies
of rows that the kernels cannot load, and the workspaces that calls ask for."""
import pytest
import torch

from breeze_amd import attention as att
from breeze_amd import hip_backend as hb


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


def _attention_bytes(kv_heads, page, D, T, B, heads, dtype, cols, has_cu=1):
    n = hb._lib.i4_paged_attention_workspace(kv_heads, page, D, T, B, heads, dtype, cols, has_cu)
    assert n >= 0, hb.last_error()
    return n


# Tables of 131072 keys.  None has room for copies in 4 GiB but the first (512 MiB + 8 MiB).
@pytest.mark.parametrize("kv_heads,D,T,B,heads,dtype,most", [
    (8, 128, 4096, 1, 32, 2, 0.9), (4, 256, 8192, 33, 24, 0, 1), (8, 128, 8192, 8, 32, 1, 1),
    (8, 128, 8192, 32, 32, 1, 1), (8, 128, 16384, 2, 64, 1, 2), (8, 128, 16384, 100, 64, 1, 1),
    (8, 128, 2048, 2048, 64, 1, 1)])
def test_workspaces_of_wide_tables(kv_heads, D, T, B, heads, dtype, most):
    """Single tokens beside chunks: the tokens' splits are no cause to keep partial sums
    of the chunks' rows."""
    assert _attention_bytes(kv_heads, 16, D, T, B, heads, dtype, 131072 // 16) <= most * 2 ** 30


def test_workspaces_have_a_bound():
    """4 GiB of copies and 512 MiB of partial sums for each kind of kernel, whatever the
    call; where a call has more rows than that, its keys are not split."""
    for D in (64, 128, 256):
        for kv_heads, heads in ((1, 1), (1, 128), (4, 24), (8, 32), (32, 32), (8, 128)):
            for T in (1, 2, 63, 64, 1000, 8192, 65536, 1 << 20):
                for B in (1, 2, 7, 64, 1000):
                    for keys in (16, 1000, 4096, 131072, 1 << 22):
                        for dtype in (0, 1):
                            if B <= T and T * heads <= 1 << 26:
                                n = _attention_bytes(kv_heads, 16, D, T, B, heads, dtype, -(-keys // 16), 1)
                                assert n <= 5 << 30, (D, kv_heads, heads, T, B, keys)
        for B in (1, 64, 4096, 32768):
            assert _attention_bytes(8, 16, D, B, B, 64, 1, 1 << 16, 0) <= 512 << 20


def test_workspaces_of_long_prompts():
    """Gated linear attention holds 1 GiB of chunks' operands at a time."""
    query = hb._lib.i4_gated_linear_attention_workspace
    for k_heads, v_heads, k_dim, v_dim in ((16, 48, 128, 128), (1, 1, 64, 16), (32, 32, 128, 256), (64, 256, 128, 128)):
        for T in (17, 1000, 4096, 40000, 131072, 1 << 20):
            for B in (1, 7, 1000):
                for dtype in (0, 1, 2):
                    for beta in (0, 1):
                        assert 0 < query(T, B, k_heads, v_heads, k_dim, v_dim, dtype, 1, beta) <= 1 << 30
    # A call of fewer operands holds them all: 25 chunks' slots of 2 times 64 KB and 6 times 25 KB.
    assert query(1536, 1, 2, 6, 128, 128, 0, 1, 1) == 25 * (2 * 65536 + 6 * 25600)
