"""Verification over the widest vocabularies: rows of more than 128 pieces of 2048
scores, up to all 1024, against the rule as it is told."""
import pytest
import torch

from drafts_plain import cu_of, walk

pytestmark = pytest.mark.gpu

LAST = 1 - 2.0 ** -24  # the largest fp32 below one
TREES = [[-1, 0, 0, 2], [-1, 0], [-1]]


@pytest.fixture
def drafts(gpu):
    from breeze_amd import drafts
    return drafts


@pytest.mark.parametrize("V", [2048 * 128, 2048 * 128 + 1, 300001, 1 << 21])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("where", ["early", "late", "anywhere"])
def test_wide(drafts, where, draft, V):
    """Top scores, children and drawn tokens in the first pieces, past the 128th (where there are
    any), or all over the row, which is flat then."""
    gen = torch.Generator().manual_seed(V % 1000 + draft)
    T = sum(len(t) for t in TREES)
    logits = 0.5 * torch.randn((T, V), generator=gen)
    lo, hi = {"early": (0, 2048), "late": (2048 * 127 + 2000, V), "anywhere": (0, V)}[where]
    tops = torch.randint(lo, hi, (T, 6), generator=gen)
    if where != "anywhere":
        logits.scatter_(1, tops, 16 + 4 * torch.rand((T, 6), generator=gen))
    q = torch.softmax(logits + 0.5 * torch.randn((T, V), generator=gen), -1) if draft else None
    tokens = torch.zeros((T,), dtype=torch.int32)
    start = 0
    for t in TREES:
        for i, p in enumerate(t):
            tokens[start + i] = int(tops[start + max(p, 0), i])
        start += len(t)
    tokens[3] = int(logits[2].argmax())
    parents, cu = torch.tensor([p for t in TREES for p in t], dtype=torch.int32).cuda(), cu_of([4, 2, 1]).cuda()
    on = logits.cuda()
    qc = None if q is None else q.cuda()
    for first, others in ((0.3, 0.5), (0.0, LAST), (LAST, LAST), (0.999, 0.0), (0.62, 0.02)):
        u = torch.full((T,), others)
        u[[0, 4, 6]] = first
        for temps in ([0.8, 1.0, 1.3], [0.0, 0.0, 0.0]):
            got = drafts.verify(on, tokens.cuda(), parents, u.cuda(), cu, torch.tensor(temps).cuda(), qc)
            new, path, counts = (x.cpu().tolist() for x in got)
            start = 0
            for b, t in enumerate(TREES):
                n = len(t)
                own = slice(start, start + n)
                # A float32's value: the kernel is given that.
                tau = float(torch.tensor(temps[b]))
                want, nodes = walk(logits[own], tokens[own], t, u[own], tau, None if q is None else q[own])
                rest = [-1] * (n - len(nodes))
                assert counts[b] == len(nodes) and path[own] == nodes + rest and new[own] == want + rest, (first, temps, b)
                start += n
