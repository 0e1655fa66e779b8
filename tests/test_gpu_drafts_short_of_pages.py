"""Steps with drafted tokens in which the free pages do not suffice: a sequence that
got none has no token, keeps its length and pages, and goes on once others have given
pages back."""
import pytest
import torch

from drafts_plain import cu_of, tree, walk
from test_gpu_drafts_together import PAGE, V, _i32, _plainly, _prompt, setup  # noqa: F401

pytestmark = pytest.mark.gpu

N = 7  # nodes of a tree


def _step(m, drafts, tokens, lens, cu, parents, uniforms, temps):
    slots, positions, kv = m.pages.extend(lens, cu, tokens.shape[0], parents)
    logits = m.forward(drafts, tokens, slots, positions, kv, cu, parents)
    new, path, counts = drafts.verify(logits, tokens, parents, uniforms, cu, temps, kv_lens=kv)
    after = drafts.kv_compact(m.caches, m.pages.table, kv, cu, path, counts, lens)
    m.pages.trim(after)
    return new, path, counts, after, kv


def _steps(m, drafts, want, step, lens, last):
    """`step` (tokens, parents, cu -> lists) over trees that hold coming tokens; sequence 2 leaves
    once the others have waited twice.  (tokens of each sequence, what each step gave)."""
    out, waited, gone, log = [[] for _ in want], 0, False, []
    for s in range(14):
        tokens, parents = [], []
        for b in range(3):
            t, p, at, good = [last[b]], [-1], 0, (s + b) % 4
            for d in range(3):
                w = want[b][len(out[b]) + d]
                wrong = (w + 1 + d) % V
                t += [wrong, w if d < good else (wrong + 5) % V]
                p += [at, at]
                at = len(t) - 1
            tokens += t
            parents += p
        new, path, counts, after, kv, held = step(tokens, parents, [0, N, 2 * N, 2 * N if gone else 3 * N], gone)
        log.append((new, path, counts, after, kv, held))
        for b in range(3):
            own, c = slice(b * N, b * N + N), counts[b]
            if b == 2 and gone:
                assert c == 0 and after[b] == 0 and held[b] == 0
            elif kv[b] < 0:
                assert c == 0 and new[own] == path[own] == [-1] * N
                assert after[b] == lens[b] and held[b] == -(-lens[b] // PAGE)
                waited += 1
            else:
                assert kv[b] == lens[b] + N and c == 1 + (s + b) % 4 and after[b] == lens[b] + c
                out[b] += new[own][:c]
                last[b] = out[b][-1]
        lens = after
        if waited >= 2 and not gone:
            gone, lens = True, after[:2] + [0]
        if min(len(out[0]), len(out[1])) > 16:
            break
    assert waited >= 2 and gone and sum(k[4][0] >= 0 for k in log[-2:]) == 2
    return out, log


def _run(make, drafts, captured):
    want = _plainly(make(3), drafts, 24)
    m = make(3, 4)  # three pages hold the prompts
    lens, last = _prompt(m, drafts)
    state, temps = lens.clone(), torch.zeros(3, device="cuda")
    held = [torch.zeros(3 * N, dtype=torch.int32, device="cuda"), torch.full((3 * N,), -1, dtype=torch.int32, device="cuda"),
            cu_of([N] * 3).cuda()]
    u = torch.rand((3 * N,), generator=torch.Generator().manual_seed(4)).cuda()
    if captured:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):  # sizes the stream's scratch of the projections; slots of -1 write nothing
            none = torch.full((3 * N,), -1, dtype=torch.int32, device="cuda")
            m.forward(drafts, held[0], none, none, torch.zeros(3, dtype=torch.int32, device="cuda"), held[2], none)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _step(m, drafts, held[0], state, held[2], held[1], u, temps)
            state.copy_(got[3])

    def step(tokens, parents, cu, gone):
        if gone:
            state[2] = 0
            m.pages.trim(state)
        for a, b in zip(held, (tokens, parents, cu)):
            a.copy_(torch.tensor(b, dtype=torch.int32))
        if captured:
            graph.replay()
            now = got
        else:
            now = _step(m, drafts, held[0], state, held[2], held[1], u, temps)
            state.copy_(now[3])
        torch.cuda.synchronize()
        return [x.tolist() for x in now] + [m.pages.held.tolist()]

    out, log = _steps(m, drafts, want, step, lens.tolist(), last)
    for o, w in zip(out, want):
        assert o == w[:len(o)]
    assert len(out[0]) > 16 and len(out[1]) > 16
    return log


def test_a_sequence_waits_for_pages(setup):  # noqa: F811
    make, att, drafts = setup
    assert _run(make, drafts, False) == _run(make, drafts, True)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_verify_passes_over_them(gpu, temperature, draft):
    """The others' tokens and paths are those without them."""
    from breeze_amd import drafts
    gen = torch.Generator().manual_seed(1)
    trees = [tree(n, gen) for n in (5, 0, 9, 1, 30, 4)]
    lens = [len(t) for t in trees]
    T, W = sum(lens), 3001
    logits = 3 * torch.randn((T, W), generator=gen)
    q = torch.softmax(logits + torch.randn((T, W), generator=gen), -1) if draft else None
    tokens, u = torch.randint(0, W, (T,), generator=gen, dtype=torch.int32), torch.rand((T,), generator=gen)
    kv = [-1, 3, 40, -2 ** 31, -7, 0]
    got = drafts.verify(logits.cuda(), tokens.cuda(), _i32([p for t in trees for p in t]), u.cuda(), cu_of(lens).cuda(),
                        temperature, None if q is None else q.cuda(), kv_lens=_i32(kv))
    new, path, counts = (x.tolist() for x in got)
    start = 0
    for b, t in enumerate(trees):
        own = slice(start, start + len(t))
        want, nodes = ([], []) if kv[b] < 0 or not t else walk(
            logits[own], tokens[own], t, u[own], float(torch.tensor(temperature)), None if q is None else q[own])
        rest = [-1] * (len(t) - len(nodes))
        assert counts[b] == len(nodes) and new[own] == want + rest and path[own] == nodes + rest
        start += len(t)
    # One node a sequence.
    got = drafts.verify(logits[:3].cuda(), tokens[:3].cuda(), None, u[:3].cuda(), kv_lens=_i32([4, -1, 0]))
    assert got[2].tolist() == [1, 0, 1] and got[0].tolist()[1] == -1 and got[1].tolist() == [0, -1, 0]


@pytest.mark.parametrize("layers", [1, 33])
def test_compaction_keeps_their_lengths(gpu, layers):
    from breeze_amd import attention as att, drafts
    gen = torch.Generator().manual_seed(2)
    caches = [att.KVCache(*(torch.randint(-9, 9, (6, 1, 16, 64), dtype=torch.int8, generator=gen).cuda() for _ in range(2)),
                          *(torch.rand((6, 1, 16), generator=gen).cuda() for _ in range(2))) for _ in range(layers)]
    table, cu = _i32([[0, 1], [2, 3], [4, 5]]), cu_of([4, 4, 4]).cuda()
    path, before = _i32([0, 2, 3, -1] * 3), _i32([5, 20, -1])
    first = [c.k.clone() for c in caches]
    args = (_i32([9, -1, -1]), cu, path, _i32([3, 3, 0]))
    got = drafts.kv_compact(caches, table, *args, before)
    assert got.tolist() == [8, 20, -1] and before.tolist() == [5, 20, -1]
    assert all(torch.equal(c.k[2:], k[2:]) and torch.equal(c.k[0, :, 6], k[0, :, 7]) for c, k in zip(caches, first))
    assert drafts.kv_compact(caches, table, *args).tolist() == [8, -1, -1]
