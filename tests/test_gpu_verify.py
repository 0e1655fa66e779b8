"""Drafted tokens against the target's logits: the walk and the drawn token
against the rule as it is told, in 64 bits, and the distribution it leaves."""
import math

import pytest
import torch

from drafts_plain import cu_of, tree, walk

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LAST = 1 - 2.0 ** -24  # the largest fp32 below one


@pytest.fixture
def drafts(gpu):
    from breeze_amd import drafts
    return drafts


def _inputs(gen, trees, V, dtype, draft, spread=3.0):
    """Scores in which a few tokens stand out, tokens that the scores (or the draft) favour."""
    T = sum(len(t) for t in trees)
    logits = spread * torch.randn((T, V), generator=gen)
    for _ in range(min(3, V)):
        logits.scatter_add_(1, torch.randint(V, (T, 1), generator=gen), 8 * torch.rand((T, 1), generator=gen))
    logits = logits.to(DT[dtype])
    rough = logits.float() + 0.8 * torch.randn((T, V), generator=gen)
    q = torch.softmax(rough, -1) if draft else None
    if draft:  # drawn without replacement
        rough = rough - torch.log(-torch.log(torch.rand((T, V), generator=gen).clamp(1e-7, 1 - 1e-7)))
    best = rough.topk(min(5, V), -1).indices
    tokens, start = [], 0
    for t in trees:
        kids = {}
        for i, p in enumerate(t):
            k = kids[p] = kids.get(p, -1) + 1
            tokens.append(int(best[start + p, k % best.shape[1]]) if p >= 0 else 0)
        start += len(t)
    return logits, torch.tensor(tokens, dtype=torch.int32), torch.rand((T,), generator=gen), q


def _call(drafts, logits, tokens, trees, uniforms, temperature, q, lens=None):
    gpu = lambda x: None if x is None else x.cuda()  # noqa: E731
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32)
    t = temperature.cuda() if isinstance(temperature, torch.Tensor) else temperature
    got = drafts.verify(logits.cuda(), gpu(tokens), gpu(parents), gpu(uniforms),
                        cu_of([len(x) for x in trees]).cuda(), t, gpu(q))
    return [x.cpu().tolist() for x in got]


def _check(drafts, logits, tokens, trees, uniforms, temperature, q):
    got, path, counts = _call(drafts, logits, tokens, trees, uniforms, temperature, q)
    start = 0
    for b, t in enumerate(trees):
        n, end = len(t), start + len(t)
        if n:
            tau = float(temperature[b]) if isinstance(temperature, torch.Tensor) else float(torch.tensor(temperature))
            new, nodes = walk(logits[start:end], tokens[start:end], t, uniforms[start:end], tau,
                              None if q is None else q[start:end])
            m = len(nodes)
        else:
            new, nodes, m = [], [], 0
        assert counts[b] == m, (b, counts[b], nodes)
        assert path[start:end] == nodes + [-1] * (n - m), b
        assert got[start:end] == new + [-1] * (n - m), (b, got[start:end], new)
        start = end
    return counts


SIZES = [1, 2, 5, 13, 0, 33, 1, 64, 7]


@pytest.mark.parametrize("V", [1, 2, 77, 2047, 2048, 2049, 5000, 32003])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("draft", [False, True])
def test_trees(drafts, draft, dtype, V):
    gen = torch.Generator().manual_seed(V + draft)
    trees = [tree(n, gen) for n in SIZES]
    logits, tokens, uniforms, q = _inputs(gen, trees, V, dtype, draft)
    temps = torch.tensor([0.7, 1.0, 0.0, 0.3, 1.0, 1.3, 1.0, 0.8, 0.0])
    _check(drafts, logits, tokens, trees, uniforms, temps, q)


@pytest.mark.parametrize("draft", [False, True])
def test_chains_of_a_wide_vocabulary(drafts, draft):
    gen = torch.Generator().manual_seed(4)
    trees = [tree(n, gen, chain=True) for n in (1, 4, 8, 6, 8, 3, 5, 8)]
    logits, tokens, uniforms, q = _inputs(gen, trees, 151936, "fp32", draft)
    _check(drafts, logits, tokens, trees, uniforms, 0.8, q)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [500, 60001])
def test_paths_that_go_down(drafts, V, draft, dtype):
    """Scores in which a node's children hold most of the weight: long paths."""
    gen = torch.Generator().manual_seed(V + 2 * draft)
    trees = [tree(n, gen, chain=n > 40) for n in (20, 60, 9, 33, 64, 12)]
    logits, tokens, uniforms, q = _inputs(gen, trees, V, dtype, draft)
    start = 0
    for t in trees:
        for i, p in enumerate(t):
            if p >= 0:
                logits[start + p, tokens[start + i]] = 24.0 - 2.0 * torch.rand((1,), generator=gen)
        start += len(t)
    if draft:
        q = torch.softmax(logits.float() + 0.5 * torch.randn(logits.shape, generator=gen), -1)
    temps = torch.tensor([1.0, 0.7, 0.5, 1.0, 0.8, 0.0])
    assert max(_check(drafts, logits, tokens, trees, uniforms, temps, q)) > 3


@pytest.mark.parametrize("draft", [False, True])
def test_flat_scores(drafts, draft):
    """Every token alike: borders as close as they get."""
    gen = torch.Generator().manual_seed(5)
    trees = [tree(5, gen)] * 20
    logits, tokens, uniforms, q = _inputs(gen, trees, 40000, "fp32", draft, spread=0.01)
    _check(drafts, logits * 0.01, tokens, trees, uniforms, 1.0, q)


@pytest.mark.parametrize("draft", [False, True])
def test_many_siblings_are_rejected(drafts, draft):
    """A root of 200 children, most of whose tokens have next to no weight; repeated tokens,
    tokens outside the vocabulary."""
    gen = torch.Generator().manual_seed(6)
    V, trees = 4100, [[-1] + [0] * 200, [-1] + [0] * 40]
    logits, _, uniforms, _ = _inputs(gen, trees, V, "fp32", False)
    tokens = torch.randint(0, V, (242,), generator=gen).to(torch.int32)
    tokens[50:80] = tokens[20:50]
    tokens[81], tokens[82], tokens[210] = -1, V, 1 << 30
    q = None
    if draft:
        q = torch.softmax(torch.randn((242, V), generator=gen), -1)
    _check(drafts, logits, tokens, trees, uniforms, 1.0, q)


def test_all_weight_on_rejected_tokens(drafts):
    """What is left is far below the rejected tokens' rounding: the sums are taken anew."""
    V = 3000
    logits = torch.full((4, V), -30.0) + torch.arange(V) * 1e-3
    logits[:, 7] = 0.0
    logits[:, 2500] = -16.0
    tokens = torch.tensor([0, 7, 2500, 9], dtype=torch.int32)
    for u in (0.0, 0.3, 0.999, LAST):
        uniforms = torch.tensor([u, LAST, LAST, LAST])
        # p(7) is 1 - 3e-8 or so above: only with more temperature is it rejected.
        for tau in (1.0, 1.2, 1.5, 2.0):
            _check(drafts, logits, tokens, [[-1, 0, 0, 0]], uniforms, tau, None)


def test_random_numbers_at_the_ends(drafts):
    """0 takes the first token that has any weight, and any child that has; the largest
    number below one the last."""
    logits = torch.full((6, 5000), -math.inf)
    logits[:, 1234:4000] = torch.randn((6, 2766), generator=torch.Generator().manual_seed(7))
    tokens = torch.tensor([0, 3, 1500, 0, 3, 1500], dtype=torch.int32)
    uniforms = torch.tensor([0.0, 0.0, LAST, LAST, LAST, LAST])
    trees = [[-1, 0, 0], [-1, 0, 0]]
    _check(drafts, logits, tokens, trees, uniforms, 1.0, None)
    got, _, counts = _call(drafts, logits, tokens, trees, uniforms, 1.0, None)
    assert counts == [1, 1] and got[0] == 1234 and got[3] == 3999  # weightless children, then the ends


def test_greedy_takes_the_first_of_equals(drafts):
    logits = torch.zeros((6, 9000))
    logits[0, [800, 8999]] = 2.0
    logits[1, [3, 2]] = 1.0
    logits[3] = -math.inf
    logits[3, 5000:] = -1.0
    tokens = torch.tensor([0, 8999, 800, 5, 5000, 5001], dtype=torch.int32)
    trees = [[-1, 0, 0], [-1, 0, 0]]
    got, path, counts = _call(drafts, logits, tokens, trees, torch.full((6,), LAST), 0.0, None)
    assert got == [800, 0, -1, 5000, 0, -1] and path == [0, 2, -1, 0, 1, -1] and counts == [2, 2]
    q = torch.full((6, 9000), 1.0 / 9000)
    assert _call(drafts, logits, tokens, trees, torch.full((6,), LAST), 0.0, q) == [got, path, counts]


@pytest.mark.parametrize("bad", ["nan", "inf", "nothing", "negative", "not a number", "infinite"])
@pytest.mark.parametrize("draft", [False, True])
def test_no_distribution(drafts, bad, draft):
    """The sequence ends there with -1; the others go on."""
    gen = torch.Generator().manual_seed(8)
    trees = [[-1, 0, 1], [-1, 0, 1], [-1]]
    logits, tokens, uniforms, q = _inputs(gen, trees, 3001, "fp32", draft)
    tokens[1] = int(logits[0].argmax())
    uniforms[1] = 0.0  # the first chain's first token is taken
    temps = torch.tensor([0.9, 0.9, 0.9])
    if bad == "nothing":
        logits[1] = -math.inf
    elif bad in ("nan", "inf"):
        logits[1, 2999] = float(bad)
    else:
        temps[0] = {"negative": -0.1, "not a number": math.nan, "infinite": math.inf}[bad]
    _check(drafts, logits, tokens, trees, uniforms, temps, q)
    got, path, counts = _call(drafts, logits, tokens, trees, uniforms, temps, q)
    if bad in ("nan", "inf", "nothing"):
        assert got[:3] == [int(tokens[1]), -1, -1] and path[:3] == [0, 1, -1]
    else:
        assert got[:3] == [-1, -1, -1] and counts[0] == 1


def test_drafts_that_are_no_distribution(drafts):
    gen = torch.Generator().manual_seed(9)
    trees = [[-1, 0], [-1, 0], [-1, 0, 0], [-1, 0, 0]]
    logits, tokens, uniforms, q = _inputs(gen, trees, 2500, "fp32", True)
    uniforms[[1, 3, 5, 6, 8, 9]] = LAST
    # Rows of nodes without children are not read.
    q[1], q[3], q[5:7], q[8:10] = math.nan, math.inf, math.nan, -1.0
    logits[0], q[0] = 0.0, 0.0
    tokens[1] = 11
    q[0, 11] = 1.0  # rejected: what is left is all but token 11
    q[2, 17] = math.nan
    tokens[3] = 12
    logits[2], q[2, 12] = 0.0, 1.0  # rejected: a draft of NaN gives no token
    # The draft leaves nothing for the second child: it is passed over.
    logits[4], q[4] = 0.0, 0.0
    tokens[5], tokens[6], q[4, 20] = 20, 21, 1.0
    # The draft gives its child no chance at all, the target some: taken.
    logits[7], q[7] = 0.0, 0.0
    tokens[8], q[7, 40] = 30, 1.0
    got, path, counts = _call(drafts, logits, tokens, trees, uniforms, 1.0, q)
    assert counts == [1, 1, 1, 2] and got[2] == -1
    for start, t in ((0, trees[0]), (4, trees[2]), (7, trees[3])):
        n = len(t)
        new, nodes = walk(logits[start:start + n], tokens[start:start + n], t, uniforms[start:start + n], 1.0,
                          q[start:start + n])
        assert got[start:start + len(new)] == new


@pytest.mark.parametrize("draft", [False, True])
def test_tokens_are_distributed_as_the_target(drafts, draft):
    """40000 sequences of one tree each; children fixed, or drawn from the draft without
    replacement.  Each token's frequency lies within five deviations of its chance."""
    gen = torch.Generator().manual_seed(10)
    B, V, n = 40000, 12, 4
    row = torch.randn((V,), generator=gen) * 1.5
    p = torch.softmax(row.double() / 0.9, 0)
    logits = row.expand(B * n, V)
    q = None
    if draft:
        q1 = torch.softmax(row + torch.randn((V,), generator=gen), 0)
        drawn = torch.multinomial(q1.expand(B, V), 3, generator=gen)
        q = q1.expand(B * n, V)
    else:
        drawn = row.topk(4).indices[1:].expand(B, 3)
    tokens = torch.cat([torch.zeros((B, 1), dtype=torch.int64), drawn], 1).to(torch.int32).reshape(-1)
    uniforms = torch.rand((B * n,), generator=gen)
    got, path, counts = _call(drafts, logits, tokens, [[-1, 0, 0, 0]] * B, uniforms, 0.9, q)
    first = torch.tensor(got).view(B, n)[:, 0]
    freq = torch.bincount(first, minlength=V).double() / B
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all(), (freq, p)
    # Where a child was taken, the token after it is the target's as well.
    second = torch.tensor(got).view(B, n)[:, 1]
    second = second[torch.tensor(counts) > 1]
    freq = torch.bincount(second, minlength=V).double() / len(second)
    assert len(second) > 5000 and ((freq - p).abs() <= 5 * (p * (1 - p) / len(second)).sqrt()).all()


def test_sizes_of_trees_and_rows_outside(drafts):
    gen = torch.Generator().manual_seed(11)
    V = 65
    trees = [tree(1024, gen, chain=True), tree(1025, gen)]
    logits, tokens, uniforms, _ = _inputs(gen, trees, V, "fp32", False)
    for i in range(1, 1024):
        tokens[i] = int(logits[i - 1].argmax())
    got, path, counts = _call(drafts, logits, tokens, trees, uniforms, 0.0, None)
    assert counts == [1024, 0] and path[:1024] == list(range(1024)) and path[1024:] == [-1] * 1025
    assert got[:1023] == tokens[1:1024].tolist() and got[1023] == int(logits[1023].argmax())
    assert got[1024:] == [-1] * 1025
    cu = torch.tensor([2, 5, 6], dtype=torch.int32).cuda()
    parents = torch.tensor([-1, -1, -1, 0, 1, -1, -1, -1, -1], dtype=torch.int32).cuda()
    got, path, counts = drafts.verify(logits[:9].cuda(), tokens[:9].cuda(), parents, uniforms[:9].cuda(), cu, 0.5)
    assert got[:2].tolist() == [-1, -1] and got[6:].tolist() == [-1] * 3 and path[6:].tolist() == [-1] * 3
    new, nodes = walk(logits[2:5], tokens[2:5], [-1, 0, 1], uniforms[2:5], 0.5)
    assert got[2:2 + len(new)].tolist() == new and counts.tolist() == [len(new), 1]


def test_single_tokens(drafts):
    """Without offsets every row draws its token."""
    gen = torch.Generator().manual_seed(12)
    logits, tokens, uniforms, _ = _inputs(gen, [[-1]] * 50, 3333, "fp32", False)
    got, path, counts = drafts.verify(logits.cuda(), tokens.cuda(), None, uniforms.cuda(), None, 0.7)
    tau = float(torch.tensor(0.7))
    want = [walk(logits[i:i + 1], tokens[i:i + 1], [-1], uniforms[i:i + 1], tau)[0][0] for i in range(50)]
    assert got.tolist() == want and path.tolist() == [0] * 50 and counts.tolist() == [1] * 50
    none = drafts.verify(logits[:0].cuda(), tokens[:0].cuda(), None, uniforms[:0].cuda())
    assert [x.shape[0] for x in none] == [0, 0, 0]
    none = drafts.verify(logits[:3].cuda(), tokens[:3].cuda(), torch.zeros(3, dtype=torch.int32).cuda(),
                         uniforms[:3].cuda(), torch.zeros(1, dtype=torch.int32).cuda())
    assert none[0].tolist() == [-1] * 3 and none[2].shape == (0,)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides(drafts, dtype):
    """Rows at odd strides and offsets, one row for all, a transposed tensor."""
    gen = torch.Generator().manual_seed(13)
    trees = [tree(6, gen), tree(3, gen)]
    logits, tokens, uniforms, q = _inputs(gen, trees, 2600, dtype, True)
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32).cuda()
    rest = (tokens.cuda(), parents, uniforms.cuda(), cu_of([6, 3]).cuda(), 0.9)
    want = drafts.verify(logits.cuda(), *rest, q.cuda())
    wide = torch.full((9, 2603), math.nan, dtype=DT[dtype], device="cuda")
    wide[:, 1:2601] = logits
    wq = torch.full((9, 2607), math.nan, device="cuda")
    wq[:, 3:2603] = q
    for x, y in ((wide[:, 1:2601], wq[:, 3:2603]),
                 (logits.cuda().t().contiguous().t(), q.cuda().t().contiguous().t())):
        assert all(torch.equal(a, b) for a, b in zip(drafts.verify(x, *rest, y), want))
    one = logits[:1].cuda()
    a = drafts.verify(one.expand(9, 2600), *rest)
    b = drafts.verify(one.expand(9, 2600).contiguous(), *rest)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("draft", [False, True])
def test_graph_and_streams(drafts, draft):
    gen = torch.Generator().manual_seed(14)
    trees = [tree(7, gen, chain=draft) for _ in range(5)]
    sets = [_inputs(gen, trees, 9001, "fp32", draft) for _ in range(3)]
    held_in = [None if x is None else x.cuda() for x in sets[0]]
    parents, cu = torch.tensor([p for t in trees for p in t], dtype=torch.int32).cuda(), cu_of([7] * 5).cuda()
    temps = torch.full((5,), 0.8, device="cuda")
    call = lambda x: drafts.verify(x[0], x[1], parents, x[2], cu, temps, x[3])  # noqa: E731
    torch.cuda.synchronize()
    stream, held = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        got = call(held_in)
    for s in sets + sets[:1]:
        now = [None if x is None else x.cuda() for x in s]
        for a, b in zip(held_in, now):
            if a is not None:
                a.copy_(b)
        want = call(now)
        held.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call(held_in))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("draft", [False, True])
def test_many_sequences(drafts, draft):
    """More sequences than a wave looks through at once, many of them without nodes."""
    gen = torch.Generator().manual_seed(11)
    sizes = [int(n) for n in torch.randint(-2, 5, (5000,), generator=gen).clamp_min(0)]
    sizes[0] = sizes[63] = sizes[4096] = sizes[-1] = 0
    trees = [tree(n, gen) for n in sizes]
    logits, tokens, uniforms, q = _inputs(gen, trees, 100, "fp16", draft)
    _check(drafts, logits, tokens, trees, uniforms, 0.9, q)
