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


def _told(row, tokens, u, q):
    """A root's children by the rule as it is told, in 64 bits: what a draft leaves is the sum
    over the tokens that are left."""
    r = torch.softmax(row[0].double(), 0)
    q, left = q[0].double().clone(), 1.0
    for i, x in enumerate(tokens):
        if left != left:
            return [-1], [0]
        if not left > 0:
            continue
        if not 0 <= float(q[x]) < float("inf"):
            return [-1], [0]
        if float(u[1 + i]) * float(q[x]) / left < float(r[x]):
            return [x], [0, 1 + i]
        r = (r - q / left).clamp_min(0)
        r[x] = q[x] = 0.0
        r, left = r / r.sum(), float(q.sum())
    total = torch.cumsum(r, 0)
    return [int((total > float(u[0]) * total[-1]).nonzero()[0])], [0]


def _confident(V, gen, rest):
    """A draft that gives its first token all but `rest`, and a target that does not."""
    q = torch.rand((1, V), generator=gen)
    top = torch.randperm(V, generator=gen)[:4]
    q[0, top] = 0.0
    q *= 0.3 * rest / q.sum()
    q[0, top[1:]] = rest * torch.tensor([0.4, 0.2, 0.1])
    q[0, top[0]] = 1.0 - rest
    row = torch.randn((1, V), generator=gen)
    row[0, top] = torch.log(torch.exp(row).sum()) + torch.tensor([-1.0, -1.5, -2.0, -2.5])
    return row, q, top.tolist()


@pytest.mark.parametrize("V", [300, 5000, 32003])
@pytest.mark.parametrize("rest", [1e-3, 1e-6, 1e-7, 2.0 ** -24])
def test_confident_drafts(drafts, rest, V):
    """The first child is rejected; the others, drawn from next to nothing, go by their share of it."""
    gen = torch.Generator().manual_seed(V)
    row, q, top = _confident(V, gen, rest)
    r, left = torch.softmax(row[0].double(), 0), q[0].double()
    r = (r - left).clamp_min(0)
    left[top[0]] = r[top[0]] = 0.0
    border = float(r[top[1]] / r.sum() / (left[top[1]] / left.sum()))
    assert 0.1 < border < 0.9
    u = torch.rand((64, 5), generator=gen)
    u[:, 1] = LAST
    u[:8, 2] = border * (1 - 1e-4)
    u[8:16, 2] = border * (1 + 1e-4)
    u[16:40, 2:] = LAST
    want = [_told(row, top, x, q) for x in u]
    taken = [len(nodes) > 1 for _, nodes in want]
    assert all(taken[:8]) and not any(taken[16:40])
    got = _root(drafts, row, top, u, q=q)
    for b, (tokens, nodes) in enumerate(want):
        m = len(nodes)
        # The child's own row gives the token after it: not looked at here.
        assert got[2][b] == [m] and got[1][b][:m] == nodes and got[0][b][0] == tokens[0], (b, u[b].tolist(), tokens, got[0][b])


def test_tokens_of_a_confident_draft_are_distributed_as_the_target(drafts):
    """40000 sequences, three children drawn from the draft without replacement: each token's
    frequency lies within five deviations of its chance."""
    gen = torch.Generator().manual_seed(3)
    B, V = 40000, 12
    q = torch.full((1, V), 1e-8)
    q[0, 5], q[0, 2], q[0, 7] = 1.0 - 1e-7, 6e-8, 3e-8
    row = 0.3 * torch.randn((1, V), generator=gen)
    p = torch.softmax(row[0].double(), 0)
    drawn = torch.multinomial(q.double().expand(B, V), 3, generator=gen)
    tokens = torch.cat([torch.zeros((B, 1), dtype=torch.int64), drawn], 1).to(torch.int32).reshape(-1)
    got = drafts.verify(row.cuda().expand(4 * B, V), tokens.cuda(),
                        torch.tensor([-1, 0, 0, 0] * B, dtype=torch.int32).cuda(),
                        torch.rand((4 * B,), generator=gen).cuda(), cu_of([4] * B).cuda(), 1.0, q.cuda().expand(4 * B, V))
    freq = torch.bincount(got[0].cpu().view(B, 4)[:, 0].long(), minlength=V).double() / B
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all(), (freq, p)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -0.25])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_child_whose_own_probability_is_none(drafts, at, bad):
    """The sequence ends there with -1, whatever siblings follow; one that takes an earlier child
    does not see it."""
    gen = torch.Generator().manual_seed(at)
    V = 3000
    row, top = torch.randn((1, V), generator=gen), [7, 2900, 1500]
    q = torch.softmax(row + torch.randn((1, V), generator=gen), -1)
    q[0, top[:at]] = 0.2  # more than the target gives: rejected by the largest random number, taken by 0
    q[0, top[at]] = bad
    u = torch.full((2, 4), LAST)
    u[:, 0] = 0.4
    u[1, 1] = 0.0
    for k in range(at + 1, 4):  # the child alone or the last, and with later siblings
        got = _root(drafts, row, top[:k], u[:, :k + 1], q=q)
        want = [_told(row, top[:k], x, q) for x in u]
        assert want[0] == ([-1], [0])
        assert got[2][0] == [1] and got[0][0] == [-1] * (k + 1) and got[1][0] == [0] + [-1] * k
        if at:
            assert got[2][1] == [2] and got[0][1][0] == top[0] and got[0][1][1] >= 0
        else:
            assert got[0][1] == [-1] * (k + 1)
