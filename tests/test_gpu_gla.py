"""Gated linear attention against the recurrence in 64 bits.

Two bounds, both fixed by the arithmetic.  Norms: each product's operands keep
22 bits (relative error 2^-22) and its fp32 sums of n terms err by about
sqrt(n) 2^-24, 2^-21 for n up to 128; a chunk has five products in a row, and
the recurrence does not enlarge an error (keys of norm 1, beta in 0..1, decays
up to 1), so independent errors of c chunks leave 5 sqrt(c) 2^-20 of the norm.
Single values: no sum errs by more than its n 2^-24 of the terms' size; the
five sums of a chunk have at most 2 * 128 + 3 * 64 terms, and the terms of a
column are no larger than the state's column (or a token's v) times the other
operand's norm, at most sqrt(64) for a chunk's rows together: 8 * 448 * 2^-24 a
chunk.  A half-precision output adds its own rounding."""
import math

import pytest
import torch

from mixers_plain import half_step, recur

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def _inputs(seed, lens, Hk, Hv, Dk, Dv, dtype, delta=True, fast=1.0):
    gen = torch.Generator().manual_seed(seed)
    T = sum(lens)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k, v = unit(rand(T, Hk, Dk)).to(DT[dtype]), unit(rand(T, Hk, Dk)).to(DT[dtype]), rand(T, Hv, Dv).to(DT[dtype])
    g = -fast * torch.exp(3 * torch.rand((T, Hv), generator=gen) - 3)
    beta = torch.sigmoid(2 * rand(T, Hv)) if delta else None
    state = rand(len(lens), Hv, Dk, Dv)
    return q, k, v, g, beta, state


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _check(o, S, q, k, v, g, beta, state, lens, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    want_o, want_S, size = recur(q, k, v, g, beta, state, lens, scale)
    rep = v.shape[1] // k.shape[1]
    T, start, worst = sum(lens), 0, 0.0
    o, S = o[:T].cpu().double(), S.cpu().double()
    assert torch.isfinite(o).all() and torch.isfinite(S).all()
    qn = q.cpu().double().norm(dim=-1).repeat_interleave(rep, 1)
    half = half_step(v.dtype) if v.dtype is not torch.float32 else 0.0
    tiny = torch.finfo(v.dtype).smallest_normal
    for b, n in enumerate(lens):
        if not n:
            assert torch.equal(S[b], torch.zeros_like(S[b]) if state is None else state[b].double())
            continue
        chunks = -(-n // 64)
        each = 8 * 448 * 2.0 ** -24 * chunks * size[b]  # [Hv, Dv]
        off = (S[b] - want_S[b]).abs()
        worst = max(worst, (off / each[:, None]).max().item())
        part = slice(start, start + n)
        err = each[None] * qn[part][:, :, None] * abs(scale) + half * want_o[part].abs().clamp_min(tiny)
        worst = max(worst, ((o[part] - want_o[part]).abs() / err).max().item())
        rel = 5 * math.sqrt(chunks) * 2.0 ** -20
        sn = ((S[b] - want_S[b]).norm() / size[b].norm()).item()
        on = ((o[part] - want_o[part]).norm() / (want_o[part].norm() + abs(scale) * size[b].norm() * qn[part].max())).item()
        print(f"chunks {chunks}: values {worst:.3f} of their bound, norms {sn / rel:.3f}, {on / (rel + half):.3f}",
              flush=True)
        assert sn <= rel and on <= rel + half
        start += n
    assert worst <= 1.0


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(2, 6, 128, 128), (1, 1, 64, 16), (3, 3, 64, 80), (1, 2, 128, 256)])
def test_single_tokens(att, dtype, delta, Hk, Hv, Dk, Dv):
    x = _inputs(1, [1] * 7, Hk, Hv, Dk, Dv, dtype, delta)
    o, S = att.gated_linear_attention(*_cuda(*x))
    _check(o, S, *x, [1] * 7)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(2, 6, 128, 128), (1, 1, 64, 16), (3, 3, 64, 80), (1, 2, 128, 256)])
def test_prompts_of_any_length(att, dtype, delta, Hk, Hv, Dk, Dv):
    lens = [1, 63, 64, 0, 65, 16, 17, 200, 2]
    x = _inputs(2, lens, Hk, Hv, Dk, Dv, dtype, delta)
    o, S = att.gated_linear_attention(*_cuda(*x), _cu(lens).cuda())
    _check(o, S, *x, lens)


@pytest.mark.parametrize("n", [0, 1, 5, 16, 17, 31, 64, 500])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_sequence(att, n, dtype):
    x = _inputs(3 + n, [n], 1, 3, 128, 64, dtype)
    o, S = att.gated_linear_attention(*_cuda(*x), _cu([n]).cuda())
    _check(o, S, *x, [n])
    x = (*x[:5], None)  # from zeros
    o, S = att.gated_linear_attention(*_cuda(*x), _cu([n]).cuda(), scale=-0.25)
    _check(o, S, *x, [n], -0.25)


@pytest.mark.parametrize("delta", [True, False])
def test_decays_of_any_strength(att, delta):
    """None, nearly none, strong ones, and some that drop the state."""
    lens = [150, 70]
    for fast in (0.0, 1e-6, 30.0):
        x = list(_inputs(20, lens, 1, 2, 64, 64, "fp32", delta, fast))
        if fast == 30.0:
            x[3][10], x[3][64], x[3][65], x[3][200] = -math.inf, -math.inf, -math.inf, -1e30
        o, S = att.gated_linear_attention(*_cuda(*x), _cu(lens).cuda())
        _check(o, S, *x, lens)
        one = [t[:2] if i < 5 and t is not None else t for i, t in enumerate(x)]
        one[3] = torch.tensor([[-math.inf, 0.0], [-1e30, -0.5]])
        o, S = att.gated_linear_attention(*_cuda(*one))
        _check(o, S, *one, [1, 1])


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_alike_keys_and_whole_betas(att, dtype):
    """Equal keys with beta 1 and no decay (each token takes the one before it
    off), beta 0 (nothing is written) and zero keys."""
    lens = [130]
    x = list(_inputs(30, lens, 1, 3, 64, 32, dtype))
    x[1] = x[1][:1].expand(130, 1, 64).contiguous().clone()
    x[1][100:104] = 0
    x[3] = torch.zeros(130, 3)
    x[4] = torch.ones(130, 3)
    x[4][:, 1] = 0
    x[4][70:, 2] = 0.5
    if dtype == "fp16":
        x[1] = (x[1].float() * 0.999).half()  # a norm of 1 at most after its rounding
    o, S = att.gated_linear_attention(*_cuda(*x), _cu(lens).cuda())
    _check(o, S, *x, lens)


@pytest.mark.parametrize("dtype", list(DT))
def test_queries_and_keys_of_unlike_size(att, dtype):
    """Rows down to 2^-12 of their chunk's largest: an element's error, 2^-28 of that at most
    beside its 22 bits, is 2^-16 of such a row's, of the bound's 2^-12."""
    lens = [130, 70]
    x = list(_inputs(33, lens, 2, 4, 128, 32, dtype))
    gen = torch.Generator().manual_seed(34)
    for i in (0, 1):
        x[i] = (x[i].float() * torch.exp2(-12 * torch.rand((200, 2, 1), generator=gen))).to(x[i].dtype)
    o, S = att.gated_linear_attention(*_cuda(*x), _cu(lens).cuda())
    _check(o, S, *x, lens)


def test_values_of_any_size(att):
    """Large and tiny values, in one column, one token, a whole head."""
    lens = [100, 3]
    x = list(_inputs(31, lens, 2, 2, 128, 48, "fp32"))
    x[2][:, 0, 5] *= 1e8
    x[2][:, 1] *= 1e-12
    x[2][40, 0] *= 1e3
    x[5][0, 1] *= 1e-12
    o, S = att.gated_linear_attention(*_cuda(*x), _cu(lens).cuda())
    _check(o, S, *x, lens)


def test_continued_prompts_and_steps(att):
    """A prompt in one call, in parts and token by token leave one state, each
    within the bound of the 64-bit one; the state may be updated in place."""
    n = 147
    x = _inputs(32, [n], 2, 4, 128, 64, "fp32")
    q, k, v, g, beta, state = _cuda(*x)
    for parts in ([n], [64, 83], [1, 1, 100, 45], [20, 16, 111]):
        s, outs, at = state.clone(), [], 0
        for p in parts:
            cut = slice(at, at + p)
            o, s2 = att.gated_linear_attention(q[cut], k[cut], v[cut], g[cut], beta[cut], s,
                                               None if p == 1 else _cu([p]).cuda(), state_out=s)
            assert s2 is s
            outs.append(o)
            at += p
        _check(torch.cat(outs), s, *x, [n])


@pytest.mark.parametrize("dtype", list(DT))
def test_views_and_outputs(att, dtype):
    lens = [70, 1, 30]
    Hk, Hv, D, T = 2, 4, 64, 101
    x = _inputs(33, lens, Hk, Hv, D, D, dtype)
    q, k, v, g, beta, state = _cuda(*x)
    cu = _cu(lens).cuda()
    want = att.gated_linear_attention(q, k, v, g, beta, state, cu)
    buf = torch.empty((T, (2 * Hk + Hv) * D), dtype=q.dtype, device="cuda")
    parts = [p.view(T, -1, D) for p in buf.split([Hk * D, Hk * D, Hv * D], 1)]
    for p, t in zip(parts, (q, k, v)):
        p.copy_(t)
    gb = torch.stack([g, beta], 1)  # strided gates
    got = att.gated_linear_attention(*parts, gb[:, 0], gb[:, 1], state, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty((T, Hk * D + 1), dtype=q.dtype, device="cuda")[:, 1:].view(T, Hk, D)
    odd.copy_(q)
    gt = g.t().contiguous().t()
    got = att.gated_linear_attention(odd, k, v, gt, beta, state, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.full((T, Hv, 2 * D), 3.0, dtype=q.dtype, device="cuda")
    s2 = state.clone()
    got = att.gated_linear_attention(q, k, v, g, beta, s2, cu, out=wide[:, :, D:], state_out=s2)
    assert torch.equal(wide[:, :, D:], want[0]) and (wide[:, :, :D] == 3).all() and torch.equal(s2, want[1])


def test_rows_outside_the_sequences_stay(att):
    lens = [40, 3, 100]
    x = _inputs(34, [160], 1, 2, 64, 32, "fp32")
    q, k, v, g, beta, _ = _cuda(*x)
    cu = (_cu(lens) + 7).cuda()
    out = torch.full((160, 2, 32), 9.0, device="cuda")
    state = torch.randn((3, 2, 64, 32), generator=torch.Generator().manual_seed(1)).cuda()
    _, S = att.gated_linear_attention(q, k, v, g, beta, state, cu, out=out)
    assert (out[:7] == 9).all() and (out[150:] == 9).all()
    _check(out[7:150], S, *(t[7:150] for t in x[:5]), state.cpu(), lens)
    # One sequence shorter than the buffer, and offsets that are none.
    out.fill_(9)
    _, S = att.gated_linear_attention(q, k, v, g, beta, state[:1], _cu([5]).cuda(), out=out)
    assert (out[5:] == 9).all()
    _check(out[:5], S, *(t[:5] for t in x[:5]), state[:1].cpu(), [5])
    bad = torch.tensor([1 << 30, -7, 90, 2], dtype=torch.int32).cuda()
    att.gated_linear_attention(q, k, v, g, beta, state, bad)
    torch.cuda.synchronize()


def test_repeats_bit_for_bit_on_streams_and_in_graphs(att):
    for lens in ([1] * 5, [150, 20, 3]):
        cu = None if max(lens) == 1 else _cu(lens).cuda()
        sets = [_cuda(*_inputs(40 + i, lens, 2, 4, 128, 64, "bf16")) for i in range(4)]
        want = [att.gated_linear_attention(*x, cu) for x in sets]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for i, x in enumerate(sets):
            with torch.cuda.stream(streams[i % 2]):
                got.append(att.gated_linear_attention(*x, cu))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        held, graphs, outs = [[t.clone() for t in sets[i]] for i in range(2)], [], []
        for h in held:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[0]):
                outs.append(att.gated_linear_attention(*h, cu))
            graphs.append(graph)
        for i in range(4):
            for h, j in zip(held, (i, 3 - i)):
                for d, s in zip(h, sets[j]):
                    d.copy_(s)
            torch.cuda.synchronize()
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            again = att.gated_linear_attention(*sets[i], cu)
            torch.cuda.synchronize()
            for a, j in ((outs[0], i), (outs[1], 3 - i), (again, i)):
                assert torch.equal(a[0], want[j][0]) and torch.equal(a[1], want[j][1])
