"""Attention of trees over the paged cache against a 64-bit form of it, within
the error that its products' documented precision gives each element."""
import pytest
import torch

from drafts_plain import attend_tree, cu_of, tree
from mixers_plain import half_step

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def mods(gpu):
    from breeze_amd import attention, drafts
    return attention, drafts


def _cache(att, gen, kv_lens, H, D, page, kind, spread=1.0, extra=0):
    """A cache whose used rows hold data and whose other rows hold what must not
    matter (NaN scales, e4m3 NaN bytes); table entries past the need are bad."""
    need = [(max(n, 0) + page - 1) // page for n in kv_lens]
    P, cols = sum(need) + 2, max(need + [1]) + extra
    order = torch.randperm(P, generator=gen).to(torch.int32)
    junk = torch.full((P, H, page, D), 0x7F, dtype=torch.int8)
    pages = [(junk if kind == "int8" else junk.view(torch.float8_e4m3fn)).cuda().clone() for _ in range(2)]
    cache = att.KVCache(*pages, *(torch.full((P, H, page), float("nan"), device="cuda") for _ in range(2)))
    table = torch.full((len(kv_lens), cols), 1 << 30, dtype=torch.int32)
    at = 0
    for b, (n, c) in enumerate(zip(kv_lens, need)):
        table[b, :c] = order[at:at + c]
        at += c
        if n > 0:
            j = torch.arange(n)
            slots = (table[b].long()[j // page] * page + j % page).to(torch.int32).cuda()
            k = torch.randn((n, H, D), generator=gen) * torch.exp(0.3 * spread * torch.randn((n, H, 1), generator=gen))
            v = torch.randn((n, H, D), generator=gen) * torch.exp(spread * torch.randn((n, H, 1), generator=gen))
            att.kv_write(cache, k.cuda(), v.cuda(), slots)
    return cache, table


def _check(got, q, cache, table, kv_lens, trees, scale, dtype):
    want, bound = attend_tree(q, cache, table, kv_lens, trees, scale, dtype is not torch.bfloat16)
    # One rounding to the type: half a step of the value, or of the smallest normal
    # number, below which the steps stay as wide.
    bound = bound + half_step(dtype) * (want.abs() + bound).clamp_min(torch.finfo(dtype).smallest_normal)
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any()
    is_number = ~torch.isnan(want)
    off, bound = (got - want).abs()[is_number], bound[is_number]
    assert torch.isfinite(bound).all()
    worst = (off / bound).max().item() if off.numel() else 0.0
    print(f"error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0


def _flat(trees):
    return torch.tensor([p for t in trees for p in t], dtype=torch.int32).cuda()


def _run(mods, seed, kind, dtype, heads, H, D, page, lens, ctx, chain=False, roots=1, scale=None, spread=1.0, extra=0,
         single=False):
    att, drafts = mods
    gen = torch.Generator().manual_seed(seed)
    kv_lens = [c + n for c, n in zip(ctx, lens)]
    cache, table = _cache(att, gen, kv_lens, H, D, page, kind, spread, extra)
    trees = [tree(n, gen, chain, min(roots, n)) for n in lens]
    q = (1.5 * torch.randn((sum(lens), heads, D), generator=gen)).to(DT[dtype])
    got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(),
                                _flat(trees), None if single else cu_of(lens).cuda(), scale)
    _check(got, q, cache, table, kv_lens, trees, scale or D ** -0.5, DT[dtype])


HEADS = [(24, 4, 256), (32, 8, 128), (8, 1, 64), (4, 4, 128)]


@pytest.mark.parametrize("heads,H,D", HEADS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_few_nodes(mods, kind, dtype, heads, H, D):
    """Up to 32 rows a key head: nodes around none, and contexts around a tile."""
    lens = [3, 1, 0, 4, 2, 5, 1, 3]
    _run(mods, 1, kind, dtype, heads, H, D, 16, lens, [0, 0, 7, 124, 127, 500, 130, 61])


@pytest.mark.parametrize("heads,H,D", HEADS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("page,kind", [(16, "fp8"), (128, "int8")])
def test_trees(mods, page, kind, dtype, heads, H, D):
    """Trees of all sizes beside one another: rows of several workgroups, tiles that the
    tree begins and ends in."""
    _run(mods, 2, kind, dtype, heads, H, D, page, [13, 64, 1, 33, 20, 0, 90, 31], [100, 33, 64, 0, 500, 3, 191, 1])


@pytest.mark.parametrize("heads,H,D", [(8, 1, 64), (12, 2, 128), (12, 2, 256)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("page,kind", [(16, "int8"), (64, "fp8")])
def test_some_nodes(mods, page, kind, dtype, heads, H, D):
    """33 to 64 rows a key head on the mean, some trees of fewer and some of several units."""
    _run(mods, 8, kind, dtype, heads, H, D, page, [6, 13, 1, 0, 9, 17, 2, 4], [700, 3, 64, 5, 1999, 130, 63, 0])


@pytest.mark.parametrize("chain,roots", [(True, 1), (False, 1), (False, 5)])
@pytest.mark.parametrize("heads,H,D", HEADS)
def test_large_trees(mods, heads, H, D, chain, roots):
    """Hundreds of nodes, over many tiles and splits; as a chain they are causal attention."""
    _run(mods, 3, "int8", "fp32", heads, H, D, 16, [300, 1024 if D == 64 else 129], [77, 0], chain, roots)


@pytest.mark.parametrize("heads,H,D", HEADS)
@pytest.mark.parametrize("dtype,kind", [("fp32", "int8"), ("bf16", "fp8"), ("fp16", "int8")])
def test_long_contexts(mods, heads, H, D, dtype, kind):
    """Contexts of many splits beside one of none."""
    _run(mods, 4, kind, dtype, heads, H, D, 32, [12, 3, 25], [4100, 0, 1777])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_values_of_unlike_sizes(mods, dtype, spread):
    _run(mods, 5, "int8", dtype, 8, 2, 128, 16, [40, 7], [300, 1000], spread=spread)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 4.0, 300.0])
def test_scales(mods, scale):
    _run(mods, 6, "int8", "fp32", 8, 2, 64, 16, [20, 5], [90, 400], scale=scale, extra=3)


def test_one_node_a_sequence(mods):
    """Without offsets every row is a sequence's single token, as paged_attention has it."""
    _run(mods, 7, "fp8", "fp32", 6, 2, 128, 16, [1] * 9, [0, 1, 15, 16, 31, 100, 127, 128, 700], single=True)


def test_chain_is_causal(mods):
    """The same numbers as causal attention's, within both calls' roundings."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(8)
    kv_lens, lens = [200, 77], [50, 77]
    cache, table = _cache(att, gen, kv_lens, 2, 128, 16, "int8")
    q = torch.randn((127, 8, 128), generator=gen).cuda()
    args = (cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda())
    cu = cu_of(lens).cuda()
    a = drafts.tree_attention(q, *args, _flat([tree(n, gen, chain=True) for n in lens]), cu)
    b = att.paged_attention(q, *args, cu)
    assert ((a - b).norm() / b.norm()).item() < 2e-6


def test_bad_pages_and_lengths(mods):
    """Pages outside the cache are not seen; lengths are cut to the table; trees whose first
    nodes the cache lacks; no keys at all; parents that are none."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(9)
    kv_lens = [200, 90, 64, 30]
    cache, table = _cache(att, gen, kv_lens, 2, 64, 16, "fp8")
    table[0, 3], table[0, 12], table[1, 0] = -1, 1 << 30, cache.num_pages
    lens = [20, 10, 40, 30]
    trees = [tree(n, gen) for n in lens]
    given = [200, 90, 17, 0]
    q = torch.randn((100, 4, 64), generator=gen)
    flat = _flat(trees)
    flat[25], flat[45] = 15, -9  # a parent that comes after its child, and one below -1
    trees[1][5], trees[2][15] = -1, -1
    got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(given, dtype=torch.int32).cuda(), flat,
                                cu_of(lens).cuda())
    _check(got, q, cache, table, given, trees, 64 ** -0.5, torch.float32)
    assert (got[70:] == 0).all()
    for bad in (-1, -2 ** 31):
        given[3] = bad
        got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(given, dtype=torch.int32).cuda(), flat,
                                    cu_of(lens).cuda())
        assert (got[70:] == 0).all()


def test_a_tree_that_is_too_large(mods):
    att, drafts = mods
    gen = torch.Generator().manual_seed(10)
    kv_lens, lens = [1100, 40], [1025, 8]
    cache, table = _cache(att, gen, kv_lens, 1, 64, 16, "int8")
    trees = [tree(n, gen) for n in lens]
    q = torch.randn((1033, 2, 64), generator=gen)
    got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(),
                                _flat(trees), cu_of(lens).cuda())
    assert torch.isnan(got[:1025]).all()
    _check(got[1025:], q[1025:], cache, table[1:], kv_lens[1:], trees[1:], 64 ** -0.5, torch.float32)


def test_nan_stays_with_its_rows(mods):
    """NaN in a query, and in a node's key or value: the rows that see it."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(11)
    kv_lens, lens = [70, 40], [12, 9]
    cache, table = _cache(att, gen, kv_lens, 2, 128, 16, "int8")
    trees = [tree(n, gen) for n in lens]
    q = torch.randn((21, 4, 128), generator=gen)
    q[3, 1, 5] = float("nan")
    for b, place in ((0, 58 + 2), (1, 31 + 4)):  # nodes 2 and 4
        page = int(table[b, place // 16])
        (cache.k_scale if b else cache.v_scale)[page, 1, place % 16] = float("nan")
    got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(),
                                _flat(trees), cu_of(lens).cuda())
    bad = torch.isnan(got).any(-1)
    assert bad[3, 1]
    q = q.nan_to_num(0)
    got[3, 1] = 0
    want, _ = attend_tree(q, cache, table, kv_lens, trees, 128 ** -0.5, True)
    want[3, 1] = 0
    assert torch.equal(torch.isnan(want), torch.isnan(got.cpu()))
    assert torch.isnan(want).any() and not torch.isnan(want).all()


def test_views_outputs_and_rows_outside(mods):
    """Columns of a fused projection, an output in place, rows outside every sequence."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(12)
    kv_lens, lens = [50, 33], [6, 9]
    cache, table = _cache(att, gen, kv_lens, 2, 64, 16, "fp8")
    trees = [tree(n, gen) for n in lens]
    wide = torch.randn((19, 4 * 64 + 3 * 64 + 1), generator=gen).cuda()
    parents = torch.full((19,), -1, dtype=torch.int32).cuda()
    parents[2:17] = _flat(trees)
    args = (cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), parents,
            torch.tensor([2, 8, 17], dtype=torch.int32).cuda())
    odd = wide[:, 1:257].view(19, 4, 64)  # an odd stride: copied
    out = torch.full((19, 4, 128), 7.0, device="cuda")[:, :, 64:]
    got = drafts.tree_attention(odd, *args, out=out)
    assert got is out and (out[:2] == 7).all() and (out[17:] == 7).all()
    _check(out[2:17], odd[2:17], cache, table, kv_lens, trees, 0.125, torch.float32)
    q = odd.clone()
    assert drafts.tree_attention(q, *args, out=q) is q
    assert torch.equal(q[2:17], out[2:17]) and torch.equal(q[:2], odd[:2])
    for T in (0, 3):
        none = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
        z = torch.zeros(0, dtype=torch.int32, device="cuda")
        q0 = torch.ones((T, 4, 64), device="cuda")
        got = drafts.tree_attention(q0, cache, none, z, torch.zeros(T, dtype=torch.int32, device="cuda"),
                                    torch.zeros(1, dtype=torch.int32, device="cuda"), out=q0)
        assert (got == 1).all()


def test_graph_and_streams(mods):
    """A captured call with other lengths and trees at each replay; two streams at once."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(13)
    cache, table = _cache(att, gen, [300, 300], 2, 128, 16, "int8")
    table = table.cuda()
    lens, kv = torch.tensor([300, 300], dtype=torch.int32).cuda(), [(250, 80), (33, 300), (12, 5)]
    q, parents = torch.randn((24, 8, 128), generator=gen).cuda(), torch.full((24,), -1, dtype=torch.int32).cuda()
    cu = torch.tensor([0, 12, 24], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    stream, held = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        got = drafts.tree_attention(q, cache, table, lens, parents, cu)
    for pair in kv:
        lens.copy_(torch.tensor(pair, dtype=torch.int32))
        parents.copy_(torch.tensor(tree(12, gen) + tree(12, gen), dtype=torch.int32))
        q.copy_(torch.randn((24, 8, 128), generator=gen))
        want = drafts.tree_attention(q, cache, table, lens, parents, cu)
        held.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 3:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(drafts.tree_attention(q, cache, table, lens, parents, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_in_place_is_the_same(mods):
    """Units whose rows do not fill their waves, many sequences: what lies past them is no one's."""
    att, drafts = mods
    gen = torch.Generator().manual_seed(14)
    lens = [int(n) for n in torch.randint(1, 12, (96,), generator=gen)]
    kv_lens = [n + int(k) for n, k in zip(lens, torch.randint(0, 200, (96,), generator=gen))]
    cache, table = _cache(att, gen, kv_lens, 2, 64, 16, "fp8")
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    q = torch.randn((sum(lens), 6, 64), generator=gen).cuda() * 3
    args = (cache, table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), _flat([tree(n, gen) for n in lens]).cuda(), cu)
    want = drafts.tree_attention(q, *args)
    for _ in range(4):
        own = q.clone()
        assert torch.equal(drafts.tree_attention(own, *args, out=own), want)


@pytest.mark.parametrize("dtype,kind", [("bf16", "fp8"), ("fp32", "int8")])
def test_many_sequences(mods, dtype, kind):
    """More sequences than a wave looks through at once, some without nodes, some without keys before them."""
    gen = torch.Generator().manual_seed(15)
    lens = [int(n) for n in torch.randint(0, 6, (700,), generator=gen)]
    ctx = [int(n) for n in torch.randint(0, 90, (700,), generator=gen)]
    for b in (0, 255, 256, 400, 511, 512, 699):
        lens[b], ctx[b] = [(0, 30), (3, 0), (0, 0), (2, 700), (5, 64), (1, 1), (0, 5)][b % 7]
    _run(mods, 16, kind, dtype, 4, 2, 64, 16, lens, ctx)
