"""Page tables against lists of pages, call after call."""
import pytest
import torch

from drafts_plain import Pages, cu_of, tree

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _check(pt, plain):
    count = int(pt.count.item())
    assert pt.free.tolist()[:count] == plain.free
    assert pt.held.tolist() == plain.held
    for row, want, n in zip(pt.table.tolist(), plain.table, plain.held):
        assert row[:n] == want[:n] and all(x == -1 for x in row[n:])


def _extend(pt, plain, lens, new, parents=None, single=False):
    args = (None, None) if single else (cu_of(new).cuda(), sum(new))
    flat = None if parents is None else _i32([p for t in parents for p in t])
    got = pt.extend(_i32(lens), *args, flat)
    want = plain.extend(lens, new, parents)
    for g, w, what in zip(got, want, ("slots", "positions", "kv_lens")):
        assert g.tolist() == w, what
    _check(pt, plain)
    return want[2]


def _new(att, pages, page, B, cols):
    pt = att.PageTable.empty(pages, page, B, cols)
    return pt, Pages(pt.table.tolist(), [0] * B, list(range(pages - 1, -1, -1)), page)


@pytest.mark.parametrize("B,page,most", [(1, 16, 300), (3, 16, 40), (64, 32, 90), (300, 16, 20), (1024, 16, 5),
                                         (2500, 64, 9)])
def test_steps(att, B, page, most):
    """A batch's life: prompts, trees, single tokens, shrinking, ended and new requests,
    on a cache that has no room for all of it."""
    gen = torch.Generator().manual_seed(B)
    cols = -(-3 * most // page) + 3
    pt, plain = _new(att, B * cols // 2 + 1, page, B, cols)
    lens = [0] * B
    for step in range(12):
        kind = step % 4
        if kind == 0:
            new, parents = torch.randint(0, most + 1, (B,), generator=gen).tolist(), None
        elif kind == 1:
            new = torch.randint(0, min(most, 33), (B,), generator=gen).tolist()
            parents = [tree(n, gen) for n in new]
        else:
            new, parents = [1] * B, None
        kv = _extend(pt, plain, lens, new, parents, single=kind >= 2)
        # Sequences that got their pages keep some of the new tokens; a few end.
        for b in range(B):
            if kv[b] >= 0:
                lens[b] += int(torch.randint(0, new[b] + 1, (1,), generator=gen))
        if kind != 2:
            ended = torch.rand((B,), generator=gen) < 0.2
            lens = [0 if e else n for e, n in zip(ended.tolist(), lens)]
            given = [-1 if x < 0.1 else n for x, n in zip(torch.rand((B,), generator=gen).tolist(), lens)]
            pt.trim(_i32(given))
            plain.trim(given)
            _check(pt, plain)
            lens = [n if g >= 0 else min(n, h * page) for n, g, h in zip(lens, given, plain.held)]


@pytest.mark.parametrize("new", [[0], [1], [16], [17], [2048], [2049], [20000], [0, 0, 0], [3000, 0, 1, 4097],
                                 [1] * 3000])
def test_lengths(att, new):
    """Sizes around a page, a launch's tokens and many tokens."""
    pt, plain = _new(att, 3 * len(new) + sum(new) // 16 + 5, 16, len(new), max(new) // 16 + 2)
    lens = [(7 * b) % 17 for b in range(len(new))]
    _extend(pt, plain, lens, new)
    pt.trim(_i32(lens))
    plain.trim(lens)
    _check(pt, plain)


def test_refusals_of_sequences(att):
    """No room: nothing from the first one that has none on; those that need no page go on."""
    pt, plain = _new(att, 6, 16, 5, 4)
    kv = _extend(pt, plain, [0, 0, 0, 0, 0], [16, 40, 0, 17, 1])
    assert kv == [16, 40, 0, 17, -1]  # six pages: 1 + 3 + 0 + 2
    kv = _extend(pt, plain, [5, 40, 0, 17, 0], [11, 9, 1, 15, 1])
    assert kv == [16, -1, -1, 32, -1]
    pt.trim(_i32([0, 16, -1, 17, 0]))
    plain.trim([0, 16, -1, 17, 0])
    _check(pt, plain)
    # Past the columns, of a negative length, and a tree past 1024 nodes.
    kv = _extend(pt, plain, [60, 16, 0, 17, -3], [5, 1, 1, 0, 1])
    assert kv == [-1, 17, 1, 17, -1]
    pt, plain = _new(att, 200, 16, 2, 80)
    gen = torch.Generator().manual_seed(0)
    kv = _extend(pt, plain, [0, 0], [1025, 1024], [tree(1025, gen), tree(1024, gen, chain=True)])
    assert kv == [-1, 1024]


def test_tokens_outside_sequences(att):
    pt, _ = _new(att, 10, 16, 2, 3)
    slots, positions, kv = pt.extend(_i32([3, 0]), _i32([2, 4, 5]), 8)
    assert slots.tolist() == [-1, -1, 3, 4, 16, -1, -1, -1]
    assert positions.tolist() == [0, 0, 3, 4, 0, 0, 0, 0] and kv.tolist() == [5, 1]
    # Offsets past the tokens are cut to them.
    slots, _, kv = pt.extend(_i32([0, 0]), _i32([-5, 2, 1 << 30]), 3)
    assert slots.tolist() == [0, 1, 16] and kv.tolist() == [2, 1]
    empty = att.PageTable.empty(3, 16, 0, 4)
    slots, positions, kv = empty.extend(_i32([]), _i32([0]), 2)
    assert slots.tolist() == [-1, -1] and positions.tolist() == [0, 0] and kv.shape == (0,)
    empty.trim(_i32([]))


def test_bad_parents_have_none(att):
    pt, _ = _new(att, 10, 16, 1, 3)
    _, positions, _ = pt.extend(_i32([4]), _i32([0, 6]), 6, _i32([-1, 0, 2, 5, 1, -7]))
    assert positions.tolist() == [4, 5, 4, 4, 6, 4]


def test_graph(att):
    """A step captured once: the table changes with each replay as with each call."""
    pt, plain = _new(att, 40, 16, 3, 12)
    lens, parents = _i32([0, 0, 0]), _i32([-1, 0, 0, -1, 0, -1])
    cu = _i32([0, 3, 5, 6])
    torch.cuda.synchronize()
    stream, held = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        slots, positions, kv = pt.extend(lens, cu, 6, parents)
        pt.trim(kv)
    now = [0, 0, 0]
    for step in range(8):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        held.replay()
        torch.cuda.synchronize()
        want = plain.extend(now, [3, 2, 1], [[-1, 0, 0], [-1, 0], [-1]])
        plain.trim(want[2])
        assert (slots.tolist(), positions.tolist(), kv.tolist()) == want
        _check(pt, plain)
        now = [n + m for n, m in zip(now, ((1, 2, 1), (3, 1, 0), (2, 2, 1))[step % 3])]
