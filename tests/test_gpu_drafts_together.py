"""A decoder layer's step with drafted tokens as a program runs it, between
quantized projections: pages, positions, cache writes, attention of the trees,
the LM head, verification and compaction, eagerly and from a captured graph.  At
temperature 0 it gives the tokens that a step for each token gives."""
import numpy as np
import pytest
import torch

from conftest import rng_weights
from drafts_plain import attend_tree, cu_of, tree, walk
from mixers_plain import half_step

pytestmark = pytest.mark.gpu

H, V, EPS = 256, 512, 1e-6
HQ, HC, D, ROT = 4, 2, 64, 32
PAGE, COLS = 16, 8


class Model:
    """Two layers of attention and an LM head; one cache a layer, one page table."""

    def __init__(self, hb, att, seed, B, pages):
        rng = np.random.default_rng(seed)
        self.hb, self.att, self.made = hb, att, []

        def pack(K, N):
            qw, sc, _ = rng_weights(rng, N, K, 8)
            self.made.append(hb.prepack(qw, (sc * 0.05).astype(np.float32), None, K, N, bits=8))
            return self.made[-1]

        self.qkv_n = [HQ * D, HC * D, HC * D]
        self.layers = [([pack(H, n) for n in self.qkv_n], pack(HQ * D, H)) for _ in range(2)]
        self.head = pack(H, V)
        self.norm = torch.from_numpy(1 + 0.1 * rng.standard_normal(H, dtype=np.float32)).cuda()
        self.embed = torch.from_numpy(rng.standard_normal((V, H), dtype=np.float32)).cuda()
        self.rope = att.Rotary(ROT)
        self.caches = [att.KVCache.empty(pages, PAGE, HC, D) for _ in self.layers]
        self.pages = att.PageTable.empty(pages, PAGE, B, COLS)

    def forward(self, drafts, tokens, slots, positions, kv_lens, cu, parents, log=None):
        """Logits of the new tokens; parents None: causal."""
        x, T, hb = self.embed[tokens.long().clamp_min(0)], tokens.shape[0], self.hb
        for (qkv, out), cache in zip(self.layers, self.caches):
            q, k, v = (p.view(T, -1, D) for p in hb.rmsnorm_matmul_multi(x, self.norm, EPS, qkv, self.qkv_n))
            q, k = self.att.rotary(self.rope, q, k, positions)
            self.att.kv_write(cache, k, v, slots)
            if parents is None:
                o = self.att.paged_attention(q, cache, self.pages.table, kv_lens, cu)
            else:
                o = drafts.tree_attention(q, cache, self.pages.table, kv_lens, parents, cu)
                if log is not None:
                    log.append((q, cache, o))
            x = x + hb.matmul(out, o.reshape(T, -1), H)
        return hb.matmul(self.head, hb.rmsnorm(x, self.norm, EPS), V)

    def free(self):
        for h in self.made:
            self.hb.free(h)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _step(m, drafts, tokens, lens, cu, parents, uniforms, temps, log=None):
    """One step of all sequences; (new tokens, path, counts, lens)."""
    slots, positions, kv = m.pages.extend(lens, cu, tokens.shape[0], parents)
    logits = m.forward(drafts, tokens, slots, positions, kv, cu, parents, log)
    new, path, counts = drafts.verify(logits, tokens, parents, uniforms, cu, temps)
    lens = drafts.kv_compact(m.caches, m.pages.table, kv, cu, path, counts)
    m.pages.trim(lens)
    return new, path, counts, lens, kv, logits


@pytest.fixture
def setup(gpu, hb, hi_prec):
    from breeze_amd import attention, drafts
    hb.set_hi_prec(True)
    models = []

    def make(B, pages=24):
        models.append(Model(hb, attention, 3, B, pages))
        return models[-1]

    yield make, attention, drafts
    for m in models:
        m.free()


PROMPTS = [[5, 77, 300, 4, 9, 11, 402], [1], [90] * 21]


def _prompt(m, drafts):
    """The prompts' keys but for the last token's, which is each tree's node 0."""
    n = [len(p) - 1 for p in PROMPTS]
    cu = cu_of(n).cuda()
    slots, positions, lens = m.pages.extend(_i32([0] * 3), cu, sum(n))
    m.forward(drafts, _i32([t for p in PROMPTS for t in p[:-1]]), slots, positions, lens, cu, None)
    return lens, [p[-1] for p in PROMPTS]


def _plainly(m, drafts, steps):
    """Greedy tokens, one a step, by causal attention."""
    lens, last = _prompt(m, drafts)
    out = [[] for _ in PROMPTS]
    for _ in range(steps):
        slots, positions, kv = m.pages.extend(lens)
        logits = m.forward(drafts, _i32(last), slots, positions, kv, None, None)
        last = logits.argmax(-1).tolist()
        lens = kv
        for o, t in zip(out, last):
            o.append(t)
    return out


def test_greedy_steps_give_the_plain_tokens(setup):
    """Trees that hold the coming tokens, wrong ones beside them: as many steps as it takes, in
    the plain order, and every call within its own tests' bounds."""
    make, att, drafts = setup
    want = _plainly(make(3), drafts, 24)
    m = make(3)
    lens, last = _prompt(m, drafts)
    gen = torch.Generator().manual_seed(1)
    out, taken = [[] for _ in PROMPTS], 0
    for step in range(8):
        tokens, trees = [], []
        for b in range(3):
            # A chain of right tokens, which a wrong one may cut, below wrong siblings.
            t, p, at, good = [last[b]], [-1], 0, (step + b) % 4
            for d in range(3):
                wrong = (want[b][len(out[b]) + d] + 1 + d) % V
                right = want[b][len(out[b]) + d] if d < good else (wrong + 5) % V
                t += [wrong, right]
                p += [at, at]
                at = len(t) - 1
            tokens.append(t)
            trees.append(p)
        cu, flat = cu_of([len(t) for t in tokens]).cuda(), _i32([x for t in trees for x in t])
        log = []
        before = lens.tolist()
        new, path, counts, lens, kv, logits = _step(m, drafts, _i32([x for t in tokens for x in t]), lens, cu, flat,
                                                    torch.rand((21,), generator=gen).cuda(), 0.0, log)
        assert kv.tolist() == [n + 7 for n in before]
        start = 0
        for b in range(3):
            c = counts[b].item()
            assert c == 1 + (step + b) % 4  # the right tokens, and the drawn one
            got = new[start:start + c].tolist()
            rows = logits[start:start + 7].cpu()
            assert (got, path[start:start + c].tolist()) == walk(rows, torch.tensor(tokens[b]), trees[b],
                                                                 torch.zeros(7), 0.0)
            out[b] += got
            last[b] = got[-1]
            start += 7
            taken += c - 1
        assert lens.tolist() == [n + c for n, c in zip(before, counts.tolist())]
        assert m.pages.held.tolist() == [-(-n // PAGE) for n in lens.tolist()]
    assert taken > 20
    for o, w in zip(out, want):
        assert o == w[:len(o)]


def test_attention_of_a_step(setup):
    """Both layers' attention against its 64-bit form on the queries that it had."""
    make, att, drafts = setup
    m = make(3)
    lens, last = _prompt(m, drafts)
    gen = torch.Generator().manual_seed(2)
    trees = [tree(n, gen) for n in (9, 1, 30)]
    T = 40
    tokens = torch.randint(V, (T,), generator=gen, dtype=torch.int32).cuda()
    cu, flat, log = cu_of([9, 1, 30]).cuda(), _i32([p for t in trees for p in t]), []
    slots, positions, kv = m.pages.extend(lens, cu, T, flat)
    m.forward(drafts, tokens, slots, positions, kv, cu, flat, log)
    for q, cache, o in log:
        want, bound = attend_tree(q, cache, m.pages.table.cpu(), kv.tolist(), trees, D ** -0.5, True)
        assert ((o.cpu().double() - want).abs() <= bound + half_step(torch.float32) * want.abs() + 1e-30).all()


def test_captured_steps(setup):
    """A step with its page table, caches and lengths in one graph, replayed: the bits of the
    eager steps, at a temperature."""
    make, att, drafts = setup
    gen = torch.Generator().manual_seed(3)
    sizes = [5, 4, 7]
    cu = cu_of(sizes).cuda()
    rounds = [(torch.randint(V, (16,), generator=gen, dtype=torch.int32).cuda(),
               _i32([p for n in sizes for p in tree(n, gen)]), torch.rand((16,), generator=gen).cuda()) for _ in range(5)]
    temps = torch.tensor([0.8, 0.0, 1.1], device="cuda")
    m = make(3)
    lens, _ = _prompt(m, drafts)
    eager = []
    for tokens, parents, uniforms in rounds:
        new, path, counts, lens, kv, _ = _step(m, drafts, tokens, lens, cu, parents, uniforms, temps)
        eager.append([x.clone() for x in (new, path, counts, lens)])
    g = make(3)
    lens, _ = _prompt(g, drafts)
    held_in = [torch.zeros_like(x) for x in rounds[0]]
    state = torch.empty_like(lens)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # sizes the stream's scratch of the projections; slots of -1 write nothing
        none = torch.full((16,), -1, dtype=torch.int32, device="cuda")
        g.forward(drafts, held_in[0], none, none, torch.zeros(3, dtype=torch.int32, device="cuda"), cu, none)
    torch.cuda.synchronize()
    state.copy_(lens)
    held = torch.cuda.CUDAGraph()
    with torch.cuda.graph(held, stream=stream):
        new, path, counts, after, _, _ = _step(g, drafts, held_in[0], state, cu, held_in[1], held_in[2], temps)
        state.copy_(after)
    for (r, want) in zip(rounds, eager):
        for a, b in zip(held_in, r):
            a.copy_(b)
        held.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((new, path, counts, state), want))
    for a, b in zip(m.caches, g.caches):
        assert torch.equal(a.k, b.k) and torch.equal(a.v_scale, b.v_scale)
    assert torch.equal(m.pages.table, g.pages.table) and torch.equal(m.pages.count, g.pages.count)
