"""Accepted nodes' cache rows moved together, against the same moves in lists."""
import pytest
import torch

from drafts_plain import cu_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def mods(gpu):
    from breeze_amd import attention, drafts
    return attention, drafts


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _caches(att, gen, layers, P, H, page, D, kind):
    out = []
    for _ in range(layers):
        k, v = (torch.randint(-128, 128, (P, H, page, D), dtype=torch.int8, generator=gen).cuda() for _ in range(2))
        if kind == "fp8":
            k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
        out.append(att.KVCache(k, v, *(torch.rand((P, H, page), generator=gen).cuda() for _ in range(2))))
    return out


def _tensors(cache):
    return [cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale]


def _path(n, m, gen):
    """m of n nodes, node 0 first, in order."""
    rest = (torch.randperm(n - 1, generator=gen)[:m - 1] + 1).sort().values.tolist()
    return [0] + rest + [-1] * (n - m)


def _check(drafts, caches, table, kv_lens, lens, path, counts, single=False):
    before = [[t.cpu().clone() for t in _tensors(c)] for c in caches]
    got = drafts.kv_compact(caches if len(caches) > 1 else caches[0], table, _i32(kv_lens),
                            None if single else cu_of(lens).cuda(), _i32(path), _i32(counts))
    page, P = caches[0].page_size, caches[0].num_pages
    rows, start, want = table.tolist(), 0, []
    moves = []
    for b, (kv, n) in enumerate(zip(kv_lens, lens)):
        keep = min(max(counts[b], 0), n)
        want.append(-1 if kv < 0 else kv - n + keep)
        for i in range(keep if kv >= 0 else 0):
            src, dst = kv - n + path[start + i], kv - n + i
            if path[start + i] <= i or path[start + i] >= n or dst < 0 or src >= len(rows[b]) * page:
                continue
            ps, pd = rows[b][src // page], rows[b][dst // page]
            if 0 <= ps < P and 0 <= pd < P:
                moves.append((ps, src % page, pd, dst % page))
        start += n
    assert got.tolist() == want
    for c, old in zip(caches, before):
        new = [t.clone() for t in old]
        for ps, rs, pd, rd in moves:  # each from what was there before
            for t, o in zip(new, old):
                t[pd, :, rd] = o[ps, :, rs]
        for t, w in zip(_tensors(c), new):
            assert torch.equal(t.cpu(), w)
    return len(moves)


@pytest.mark.parametrize("kind,H,page,D", [("int8", 4, 16, 256), ("fp8", 8, 32, 128), ("int8", 1, 64, 64),
                                           ("fp8", 3, 16, 64)])
@pytest.mark.parametrize("layers", [1, 3, 33])
def test_paths(mods, kind, H, page, D, layers):
    """Trees of one to many nodes, paths of all lengths, in one launch's layers and in two."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(layers + D)
    lens = [1, 2, 5, 0, 33, 64, 17, 100]
    ctx = [0, 15, 40, 9, 3, 16, 31, 1]
    kv = [c + n for c, n in zip(ctx, lens)]
    need = [-(-n // page) for n in kv]
    P = sum(need) + 3
    order = torch.randperm(P, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    caches = _caches(att, gen, layers, P, H, page, D, kind)
    for most in (1, 4, 1000):
        path, counts = [], []
        for n in lens:
            m = int(torch.randint(1, min(n, most) + 1, (1,), generator=gen)) if n else 0
            path += _path(n, m, gen) if n else []
            counts.append(m)
        moved = _check(drafts, caches, table.cuda(), kv, lens, path, counts)
        assert most == 1 or moved > 0


def test_every_row_is_another_ones_source(mods):
    """Node i + 1 to place i, all along 300 nodes: each place is read before it is written."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(1)
    caches = _caches(att, gen, 2, 25, 2, 16, 128, "int8")
    table = torch.randperm(25, generator=gen)[:20].to(torch.int32).view(1, 20).cuda()
    path = [0] + list(range(2, 300)) + [-1]
    assert _check(drafts, caches, table, [5 + 300], [300], path, [299]) == 298


def test_what_moves_nothing(mods):
    att, drafts = mods
    gen = torch.Generator().manual_seed(2)
    caches = _caches(att, gen, 1, 6, 2, 16, 64, "int8")
    table = _i32([[0, 1], [2, 99], [4, -5], [3, 5], [1, 0], [0, 1]])
    lens = [4, 20, 20, 3, 4, 6]
    # A length of -1; pages that are not the cache's; counts outside the tree; a tree that starts
    # before the cache; numbers that are no node's, or do not grow past their place.
    kv = [-1, 25, 25, 10, 2, 12]
    path = [0, 2, 3, -1] + [0, 7, 14, 19] + [-1] * 16 + [0, 13, 15, 16] + [-1] * 16 + [0, 2, -1] + [0, 2, 3, -1]
    path += [0, 9, 1, -3, 4, 5]
    _check(drafts, caches, table, kv, lens, path, [3, 4, 4, -2, 3, 6])
    _check(drafts, caches, table, kv, lens, path, [9, 0, 30, 1 << 30, 4, 2])
    # One node a sequence.
    _check(drafts, caches, table, [3, 0, 7, -1, 1, 5], [1] * 6, [0] * 6, [1, 1, 0, 1, 1, 1], single=True)
    none = drafts.kv_compact(caches, torch.zeros((0, 3), dtype=torch.int32, device="cuda"), _i32([]), _i32([0]),
                             _i32([]), _i32([]))
    assert none.shape == (0,)


def test_graph(mods):
    att, drafts = mods
    gen = torch.Generator().manual_seed(3)
    caches = _caches(att, gen, 2, 8, 2, 16, 64, "fp8")
    table, kv, cu = _i32([[3, 1], [6, 2]]), _i32([20, 9]), _i32([0, 8, 14])
    path, counts = _i32([0] * 14), _i32([0, 0])
    torch.cuda.synchronize()
    stream, held = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        lens = drafts.kv_compact(caches, table, kv, cu, path, counts)
    for step in range(3):
        for c in caches:
            for t in _tensors(c)[:2]:
                t.copy_(torch.randint(-100, 100, t.shape, dtype=torch.int8, generator=gen))
        counts.copy_(torch.tensor([step + 1, 3 - step], dtype=torch.int32))
        path.copy_(torch.tensor(_path(8, step + 1, gen) + _path(6, 3 - step, gen), dtype=torch.int32))
        before = [[t.clone() for t in _tensors(c)] for c in caches]
        want = drafts.kv_compact(caches, table, kv, cu, path, counts)
        after = [[t.clone() for t in _tensors(c)] for c in caches]
        for c, old in zip(caches, before):
            for t, o in zip(_tensors(c), old):
                t.copy_(o)
        held.replay()
        torch.cuda.synchronize()
        assert torch.equal(lens, want)
        for c, w in zip(caches, after):
            assert all(torch.equal(t, x) for t, x in zip(_tensors(c), w))
