"""Verification where little is left: siblings that hold nearly all of a row, drafts
that give one token nearly everything."""
import pytest
import torch

from drafts_plain import cu_of, walk

pytestmark = pytest.mark.gpu

LAST = 1 - 2.0 ** -24  # the largest fp32 below one


@pytest.fixture
def drafts(gpu):
    from breeze_amd import drafts
    return drafts


def _root(drafts, row, tokens, uniforms, temperature=1.0, q=None):
    """Trees of a root and its children over one row: `uniforms` [B, 1 + children]."""
    B, n = uniforms.shape
    parents = torch.tensor(([-1] + [0] * (n - 1)) * B, dtype=torch.int32)
    given = torch.tensor(([0] + list(tokens)) * B, dtype=torch.int32)
    wide = lambda x: x.cuda().expand(B * n, -1)  # noqa: E731
    got = drafts.verify(wide(row), given.cuda(), parents.cuda(), uniforms.reshape(-1).cuda(), cu_of([n] * B).cuda(),
                        temperature, None if q is None else wide(q))
    return [x.cpu().view(B, -1).tolist() for x in got]


def _drawn(weights, u, steps):
    """The tokens that a random number may draw: those whose running sum passes it, to within
    what the sums err by.  A running sum of V terms in 64 bits errs by V 2^-53 of the whole;
    each of `steps` rejected shares that came off a sum, and their exponentials' 1.4e-14 (two
    of 7e-15), count up to 2^10 times, as a difference of less than 2^-10 is taken anew."""
    total = torch.cumsum(weights, 0)
    off = len(weights) * 2.0 ** -53 + 2.0 ** 10 * (steps * 2.0 ** -53 + 1.4e-14)
    first = lambda x: int((total > x * total[-1]).nonzero()[0])  # noqa: E731
    return first(u * (1 - off)), first(min(u * (1 + off), 1 - 2.0 ** -53))


@pytest.mark.parametrize("k,gap", [(3, 6.4), (5, 6.4), (6, 6.4), (12, 3.0), (20, 2.0), (40, 1.0), (200, 0.25)])
def test_siblings_that_each_leave_a_little(drafts, k, gap):
    """No single rejection takes most of what is left, all together leave e^(-gap k): all in one
    piece of the row, beside a flat tail of as much weight as the next sibling would have."""
    V, gen = 6000, torch.Generator().manual_seed(k)
    row = torch.full((1, V), -gap * k - 8.0)
    tokens = torch.randperm(2000, generator=gen)[:k]
    row[0, tokens] = -gap * torch.arange(k).float()
    u = torch.full((51, k + 1), LAST)
    u[:, 0] = (torch.arange(51) + 0.5) / 51
    tree = [-1] + [0] * k
    given = torch.tensor([0] + tokens.tolist())
    # The last sibling, next to its border: taken, and not.
    r = torch.softmax(row[0].double(), 0)
    r[tokens[:-1]] = 0.0
    border = float(r[tokens[-1]] / r.sum())
    u[-2, k], u[-1, k] = border * (1 - 1e-6), border * (1 + 1e-6)
    rows, whole = row.expand(k + 1, -1), torch.softmax(row[0].double(), 0)
    r[tokens[-1]] = 0.0
    new, path, counts = _root(drafts, row, tokens.tolist(), u)
    for b, x in enumerate(u):
        want, nodes = walk(rows, given, tree, x, 1.0)
        m = len(nodes)
        assert counts[b] == [m] and path[b][:m] == nodes and new[b][:m - 1] == want[:-1], (b, x.tolist())
        # From what the siblings leave, or after the one that was taken from the whole row.
        lo, hi = _drawn(r if m == 1 else whole, float(x[0]), k)
        assert lo <= want[-1] <= hi and lo <= new[b][m - 1] <= hi, (b, float(x[0]), want, new[b][:m])
        assert hi - lo <= 1  # no more than a border's two sides
