"""Which outputs of rotary positions count as lying on another tensor, against the
sets of elements, on the CPU."""
import itertools

import pytest
import torch

from breeze_amd import attention as att


def _elements(t):
    """Element numbers of a view in its storage."""
    at = t.storage_offset() + sum((torch.arange(n) * s).view([-1 if i == d else 1 for i in range(3)])
                                  for d, (n, s) in enumerate(zip(t.shape, t.stride())))
    return set(at.flatten().tolist())


def _views():
    """Views [T, heads, D] of one buffer: columns of tokens, of heads, both, with odd steps."""
    x = torch.zeros(6 * 96)
    out = []
    for T, H, D in itertools.product((1, 2, 3), (1, 2, 3), (2, 4, 8)):
        for token, head in ((96, 24), (96, 8), (96, 32), (48, 16), (40, 12), (8, 32), (24, 72), (0, 8)):
            for start in (0, 4, 8, 16, 24, 52):
                if start + (T - 1) * token + (H - 1) * head + D <= x.numel():
                    out.append(x.as_strided((T, H, D), (token, head, 1), start))
    return out


def test_disjoint_is_never_wrong():
    """Views that are said to be disjoint are; and apart ones are found so where either steps
    by whole tokens, or whole heads, of one projection."""
    views, found, truly = _views(), 0, 0
    gen = torch.Generator().manual_seed(0)
    sets = [_elements(v) for v in views]
    for i, j in torch.randint(len(views), (40000, 2), generator=gen).tolist():
        apart = not sets[i] & sets[j]
        said = att._disjoint(views[i], views[j])
        assert not said or apart, (views[i].stride(), views[i].shape, views[j].stride(), views[j].shape)
        found, truly = found + said, truly + apart
    assert found > truly / 2


@pytest.mark.parametrize("T", [1, 5])
def test_heads_that_hold_all_three(T):
    """A projection whose heads each hold q, k and v: columns of the heads."""
    x = torch.zeros((T, 4 * 3 * 64)).view(T, 4, 3, 64)
    q, k, v = x.unbind(2)
    assert att._disjoint(q, k) and att._disjoint(k, q) and att._disjoint(k, v)
    assert not att._disjoint(q, q) and not att._disjoint(q, x[:, :, 0, 2:])


def test_one_token_is_itself_whatever_its_stride():
    x = torch.zeros((3, 4 * 64))
    a, b = x[:1].view(1, 4, 64), x[0].view(1, 4, 64)
    assert att._same_rows(a, b.as_strided((1, 4, 64), (7, 64, 1))) and not att._same_rows(a, x[1].view(1, 4, 64))
    assert not att._same_rows(x.view(3, 4, 64), x.as_strided((3, 4, 64), (64, 64, 1)))
