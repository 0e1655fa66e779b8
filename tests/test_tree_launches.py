"""Tree attention's launches stay below 2^24 workgroups, whatever the sizes: calls
that would pass that are refused before anything is launched, on the CPU."""
import ctypes

import pytest

from breeze_amd import attention as att
from breeze_amd import hip_backend as hb


def _need(H, D, T, B, heads, cols, dtype=0, has_cu=1):
    return hb._lib.i4_tree_attention_workspace(H, 16, D, T, B, heads, dtype, cols, has_cu)


def test_join_of_nearly_empty_units():
    """A mean tree of 1.000001 nodes of 17 heads counts as two: units of 128 rows, one for each of
    986894 sequences, whose join would take 16 workgroups each, 17.9 million together."""
    B = 986894
    assert _need(1, 256, B + 1, B, 17, 64) == -2 and "too much" in hb.last_error()
    c = att._CCache(4096, 4096, 4096, 4096, 2, 1, 16, 256, 0)
    rc = hb._lib.i4_tree_attention_dev(ctypes.addressof(c), 4096, 4352, 256, B + 1, 17, 0, 4096, 64, 64, 4096, 4096, B, 4096,
                                       0.1, 4096, 4352, 256, None, 0, None)
    assert rc == -2 and "too much" in hb.last_error()
    # One node each: units of 32 rows.  Tables of one tile: nothing to join.
    assert _need(1, 256, B, B, 17, 64) > 0
    assert _need(1, 256, B + 1, B, 17, 4) > 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,heads", [(1, 1), (1, 17), (1, 33), (1, 65), (4, 24), (8, 136), (64, 64)])
def test_refused_by_what_is_launched(D, H, heads):
    """Sizes around the limit, counted here from the rows a unit holds."""
    for B in (1 << 10, 60000, (1 << 20) // H - 7, (1 << 20) // H):
        for T in (B, B + 1, 2 * B, 4 * B):
            if T * heads > 1 << 24 or B * H > 1 << 20:
                assert _need(H, D, T, B, heads, 1000) == -2
                continue
            G = heads // H
            mean = -(-T // B) * G
            rt = 32 if mean <= 32 else 64 if mean <= 64 and D < 256 else 128
            units = (T * G // rt + B) * H
            join = units * (rt * D // 256 // 8)
            assert (_need(H, D, T, B, heads, 1000) >= 0) == (join < 1 << 24), (B, T, join)
