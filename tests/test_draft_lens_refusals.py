"""What verification and compaction refuse of the lengths that tell them which
sequences had no place in the cache, on the CPU."""
import ctypes

import pytest
import torch

from breeze_amd import attention as att
from breeze_amd import drafts
from breeze_amd import hip_backend as hb

I32 = torch.int32


def _ints(*shape):
    return torch.zeros(shape, dtype=I32)


BAD = [_ints(3), _ints(2).long(), torch.zeros(2), _ints(2, 1), _ints(4)[::2]]


@pytest.mark.parametrize("bad", BAD)
def test_verify(bad):
    args = (torch.zeros((5, 40)), _ints(5), _ints(5), torch.zeros(5), torch.tensor([0, 2, 5], dtype=I32))
    with pytest.raises(ValueError, match="kv_lens"):
        drafts.verify(*args, kv_lens=bad)
    with pytest.raises(ValueError, match="GPU"):
        drafts.verify(*args, kv_lens=_ints(2))


@pytest.mark.parametrize("bad", BAD)
def test_kv_compact(bad):
    cache = att.KVCache.empty(3, 16, 2, 64, device="cpu")
    args = (cache, _ints(2, 2), _ints(2), torch.tensor([0, 2, 5], dtype=I32), _ints(5), _ints(2))
    with pytest.raises(ValueError, match="lens"):
        drafts.kv_compact(*args, bad)
    with pytest.raises(ValueError, match="GPU"):
        drafts.kv_compact(*args, _ints(2))


def test_c_entries():
    """The checks of the calls without the lengths, and nothing to do without sequences."""
    verify, compact = hb._lib.i4_verify_lens_dev, hb._lib.i4_kv_compact_lens_dev
    assert verify(4096, 100, 4, 0, 0, 4096, 4096, 4096, 4096, 2, 4096, None, 1.0, None, 0, 4096, 4096, 4096, None, 0, None) == -2
    assert verify(4096, 100, 4, 100, 0, 4096, 4096, 4096, 4096, 2, 4096, None, 1.0, None, 0, 4096, 4096, 4096, None, 0,
                  None) == -4
    assert verify(None, 100, 0, 100, 0, None, None, None, 4096, 0, None, None, 1.0, None, 0, None, None, None, None, 0, None) == 0
    c = att._CCache(4096, 4096, 4096, 4096, 2, 2, 16, 64, 0)
    several = (ctypes.c_void_p * 1)(ctypes.addressof(c))
    assert compact(several, 1, 4096, 1, 1, 4096, 4096, 4096, 4, 2, 4096, 4096, 4096, None) == -2
    assert compact(several, 1, 4096, 1, 1, 4096, 4096, 4096, 4, 0, 4096, 4096, 8192, None) == 0
