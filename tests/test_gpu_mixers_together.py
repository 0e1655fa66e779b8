"""The token mixers as a decoder uses them, between its quantized projections:
a linear-attention layer and a full-attention layer over two sequences, prompts
in chunks and then token by token, eagerly and from a captured graph.  Every
mixer call is checked against its 64-bit form on the inputs that it had, and a
captured step leaves the bits that the eager one does."""
import pytest
import torch

from conftest import rng_weights
from mixers_plain import attend, half_step, recur

pytestmark = pytest.mark.gpu

H, EPS = 512, 1e-6           # hidden size
HK, HV, DL = 2, 4, 64        # linear attention: key heads, value heads, their size
HQ, HC, DA = 4, 2, 64        # full attention: query heads, cached heads, their size
PAGE = 16


class Layers:
    def __init__(self, hb, seed):
        import numpy as np
        rng = np.random.default_rng(seed)
        self.hb, self.made = hb, []

        def pack(K, N):
            qw, sc, _ = rng_weights(rng, N, K, 8)
            self.made.append(hb.prepack(qw, (sc * 0.05).astype(np.float32), None, K, N, bits=8))
            return self.made[-1]

        self.lin_n = [(2 * HK + HV) * DL, HV * 16]  # q, k, v; the gates (16 columns a head, one used)
        self.lin = [pack(H, n) for n in self.lin_n]
        self.lin_out = pack(HV * DL, H)
        self.att_n = [HQ * DA, HC * DA, HC * DA]
        self.att = [pack(H, n) for n in self.att_n]
        self.att_out = pack(HQ * DA, H)
        self.norm = torch.from_numpy(1 + 0.1 * rng.standard_normal(H, dtype=np.float32)).cuda()

    def free(self):
        for h in self.made:
            self.hb.free(h)


def _step(att, layers, x, state, cache, slots, table, kv_lens, cu, log=None):
    """Both layers over packed rows x; state and cache are updated in place."""
    hb, T = layers.hb, x.shape[0]
    qkv, gates = hb.rmsnorm_matmul_multi(x, layers.norm, EPS, layers.lin, layers.lin_n)
    q, k, v = (p.view(T, -1, DL) for p in qkv.split([HK * DL, HK * DL, HV * DL], 1))
    q, k = (torch.nn.functional.normalize(p, dim=-1) for p in (q, k))
    gates = gates.view(T, HV, 16)
    g, beta = -torch.nn.functional.softplus(gates[:, :, 0]), torch.sigmoid(gates[:, :, 1])
    before = state.clone() if log is not None else None
    o, _ = att.gated_linear_attention(q, k, v, g, beta, state, cu, state_out=state)
    x = x + hb.matmul(layers.lin_out, o.reshape(T, -1), H)
    qa, ka, va = (p.view(T, -1, DA) for p in hb.rmsnorm_matmul_multi(x, layers.norm, EPS, layers.att, layers.att_n))
    att.kv_write(cache, ka, va, slots)
    oa = att.paged_attention(qa, cache, table, kv_lens, cu)
    if log is not None:
        log.append((q, k, v, g, beta, before, o, state.clone(), qa, oa, kv_lens.tolist(),
                    [1] * T if cu is None else (cu[1:] - cu[:-1]).tolist()))
    return x + hb.matmul(layers.att_out, oa.reshape(T, -1), H)


def _check(log, cache, table):
    for q, k, v, g, beta, before, o, after, qa, oa, kv, lens in log:
        want_o, want_S, size = recur(q, k, v, g, beta, before, lens, DL ** -0.5)
        # As in the operators' own tests: 8 * 448 * 2^-24 a chunk of the largest column.
        each = 8 * 448 * 2.0 ** -24 * (-(-max(lens) // 64))
        assert ((after.cpu().double() - want_S).abs() <= each * size[:, :, None] + 1e-30).all()
        rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        assert ((o.cpu().double() - want_o).abs() <= each * size[rows] * DL ** -0.5 + 2.0 ** -24 * want_o.abs()).all()
        want, bound = attend(qa, cache, table.cpu(), kv, lens, DA ** -0.5, True)
        assert ((oa.cpu().double() - want).abs() <= bound + half_step(torch.float32) * want.abs() + 1e-30).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_two_layers_in_chunks_and_steps(gpu, hb, hi_prec, kind):
    from breeze_amd import attention as att
    hb.set_hi_prec(True)
    layers = Layers(hb, 1)
    try:
        gen = torch.Generator().manual_seed(2)
        lens = [83, 21]  # prompt lengths; five steps follow
        steps = 5
        xs = [torch.randn((n + steps, H), generator=gen).cuda() for n in lens]
        cols = 7
        table = torch.randperm(2 * cols + 3, generator=gen)[:2 * cols].view(2, cols).to(torch.int32).cuda()

        def slots(b, lo, hi):
            j = torch.arange(lo, hi, device="cuda")
            return (table[b].long()[j // PAGE] * PAGE + j % PAGE).to(torch.int32)

        def run(cuts, graph=False):
            """The prompts cut at `cuts` (per call, tokens of each sequence), then steps."""
            cache = att.KVCache.empty(2 * cols + 3, PAGE, HC, DA, kind)
            state = torch.zeros((2, HV, DL, DL), device="cuda")
            log, outs, at = [], [[], []], [0, 0]
            for cut in cuts:
                x = torch.cat([xs[b][at[b]:at[b] + n] for b, n in enumerate(cut)])
                s = torch.cat([slots(b, at[b], at[b] + n) for b, n in enumerate(cut)])
                at = [a + n for a, n in zip(at, cut)]
                cu = torch.tensor([0, cut[0], cut[0] + cut[1]], dtype=torch.int32, device="cuda")
                kv = torch.tensor(at, dtype=torch.int32, device="cuda")
                y = _step(att, layers, x, state, cache, s, table, kv, cu, log)
                _check(log[-1:], cache, table)
                for b, part in enumerate(y.split(list(cut))):
                    outs[b].append(part)
            if not graph:
                for _ in range(steps):
                    x = torch.stack([xs[b][at[b]] for b in range(2)])
                    s = torch.cat([slots(b, at[b], at[b] + 1) for b in range(2)])
                    at = [a + 1 for a in at]
                    y = _step(att, layers, x, state, cache, s, table, torch.tensor(at, dtype=torch.int32).cuda(), None,
                              log)
                    _check(log[-1:], cache, table)
                    for b in range(2):
                        outs[b].append(y[b:b + 1])
            else:
                x, s = torch.zeros((2, H), device="cuda"), torch.full((2,), -1, dtype=torch.int32, device="cuda")
                kv = torch.tensor(at, dtype=torch.int32, device="cuda")
                stream = torch.cuda.Stream()
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):  # sizes the stream's scratch of the projections
                    _step(att, layers, x, state.clone(), cache, s, table, kv, None)
                torch.cuda.synchronize()
                held = torch.cuda.CUDAGraph()
                with torch.cuda.graph(held, stream=stream):
                    y = _step(att, layers, x, state, cache, s, table, kv, None)
                for _ in range(steps):
                    x.copy_(torch.stack([xs[b][at[b]] for b in range(2)]))
                    s.copy_(torch.cat([slots(b, at[b], at[b] + 1) for b in range(2)]))
                    at = [a + 1 for a in at]
                    kv.copy_(torch.tensor(at, dtype=torch.int32))
                    held.replay()
                    torch.cuda.synchronize()
                    for b in range(2):
                        outs[b].append(y[b:b + 1].clone())
            return [torch.cat(o) for o in outs], state, cache

        whole = run([tuple(lens)])
        cut = run([(40, 0), (3, 21), (40, 0)])
        held = run([tuple(lens)], graph=True)
        # One way of working through the same tokens: the same bits from the graph.
        assert torch.equal(whole[1], held[1])
        for f in ("k", "v"):
            assert torch.equal(getattr(whole[2], f).view(torch.int8), getattr(held[2], f).view(torch.int8))
        for a, b in zip(whole[0], held[0]):
            assert torch.equal(a, b)
        # Other chunks: the mixers' roundings differ, and INT16 activations make a step of
        # 2^-16 of a block's largest value out of the smallest difference; two projections
        # of the mixers' outputs and two of the rows follow one another.
        for a, b in zip(whole[0], cut[0]):
            assert ((a - b).norm() / a.norm()).item() < 4 * 2.0 ** -15
    finally:
        layers.free()
