"""Numbers that are none in gated linear attention: which rows they reach does not
depend on the form that a sequence takes, token by token or in chunks."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAN, INF = float("nan"), float("inf")


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _bad(t):
    return ~torch.isfinite(t)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
# Alone, so in chunks from 17 tokens on; beside others; and token by token.
@pytest.mark.parametrize("lens,b", [([150], 0), ([70, 150, 3], 1), ([40, 16, 20], 1)])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(2, 4, 128, 80), (1, 2, 64, 32)])
def test_a_token_reaches_its_row_and_later_ones(att, dtype, delta, value, lens, b, Hk, Hv, Dk, Dv):
    gen = torch.Generator().manual_seed(1)
    T, n, start = sum(lens), lens[b], sum(lens[:b])
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k = (unit(torch.randn((T, Hk, Dk), generator=gen)) for _ in range(2))
    v, g = torch.randn((T, Hv, Dv), generator=gen), -torch.rand((T, Hv), generator=gen)
    beta, state = torch.rand((T, Hv), generator=gen), torch.randn((len(lens), Hv, Dk, Dv), generator=gen)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    rows = sorted({0, 1, n // 2, n - 1, min(63, n - 1), min(64, n - 1), min(79, n - 1)})
    h, rep = Hv - 1, Hv // Hk
    hk = h // rep
    # Zeros in the places to be spoilt, so that they set no scale.
    for i in rows:
        q[start + i, hk, 5] = k[start + i, hk, 7] = v[start + i, h, 9] = 0.0
    q, k, v = (t.to(DT[dtype]) for t in (q, k, v))

    def run(q, k, v, g, beta):
        o, S = att.gated_linear_attention(*(t.cuda() for t in (q, k, v, g)), beta.cuda() if delta else None, state.cuda(), cu)
        return o.cpu(), S.cpu()

    clean = run(q, k, v, g, beta)
    mine = slice(start, start + n)
    heads = torch.zeros(Hv, dtype=torch.bool)
    heads[hk * rep:hk * rep + rep] = True
    for i in rows:
        for what in ("q", "k", "v", "g", "beta"):
            if what == "beta" and not delta or what == "g" and value == -INF:
                continue  # that drops the state
            x = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone(), beta=beta.clone())
            at = dict(q=(hk, 5), k=(hk, 7), v=(h, 9), g=(h,), beta=(h,))[what]
            x[what][(start + i, *at)] = value
            o, S = run(**x)
            of = heads if what in ("q", "k") else torch.arange(Hv) == h
            cols = torch.arange(Dv) == 9 if what == "v" else torch.ones(Dv, dtype=torch.bool)
            # Nothing else changes: other sequences, heads and (of v) columns, and the rows before.
            touched = torch.zeros_like(o, dtype=torch.bool)
            last = start + i + 1 if what == "q" else start + n
            touched[start + i:last] = of[:, None] & cols
            assert torch.equal(o[~touched], clean[0][~touched]), (what, i)
            others = torch.ones(len(lens), dtype=torch.bool)
            others[b] = False
            assert torch.equal(S[others], clean[1][others])
            if what == "q":
                assert torch.equal(S, clean[1])
                assert _bad(o[start + i][of]).all(), (what, i)
                continue
            keep = ~(of[:, None, None] & cols).expand(Hv, Dk, Dv)
            assert torch.equal(S[b][keep], clean[1][b][keep]), (what, i)
            # All of the rows from there on.  Token by token an infinity may leave finite
            # numbers (a key's reaches one row of the state, as does its NaN without beta);
            # in chunks all turn to NaN.
            if value != value:
                assert torch.isnan(o[mine][i:][:, of][:, :, cols]).all(), (what, i)
                assert torch.isnan(S[b][~keep]).any(), (what, i)
            if n > 16:
                assert torch.isnan(o[mine][i:][:, of][:, :, cols]).all() and torch.isnan(S[b][~keep]).all(), (what, i)


@pytest.mark.parametrize("delta", [True, False])
def test_padding_behind_a_prompt(att, delta):
    """Tokens behind a prompt's end that belong to it and hold junk: the prompt's rows are
    those without them."""
    gen = torch.Generator().manual_seed(2)
    n, pad, Hk, Hv, D = 100, 28, 2, 4, 64
    q, k = (torch.randn((n + pad, Hk, D), generator=gen).cuda() / 8 for _ in range(2))
    v, g = torch.randn((n + pad, Hv, D), generator=gen).cuda(), -torch.rand((n + pad, Hv), generator=gen).cuda()
    beta = torch.rand((n + pad, Hv), generator=gen).cuda() if delta else None
    for t in (q, k, v, g):
        t[n:] = 0
    cu = torch.tensor([0, n + pad], dtype=torch.int32).cuda()
    want, _ = att.gated_linear_attention(q, k, v, g, beta, None, cu)
    for t in (q, k, v, g) + ((beta,) if delta else ()):
        t[n:] = NAN
    got, S = att.gated_linear_attention(q, k, v, g, beta, None, cu)
    assert torch.equal(got[:n], want[:n]) and torch.isnan(got[n:]).all() and torch.isnan(S).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_large_values_that_are_finite(att, dtype):
    """Values whose sum leaves fp32, each of them finite, are no cause for NaN."""
    gen = torch.Generator().manual_seed(3)
    top = torch.finfo(DT[dtype]).max / 2
    n, D = 80, 64
    q, k = (torch.randn((n, 1, D), generator=gen) * 1e-6 for _ in range(2))
    v = torch.full((n, 2, 32), float(top))
    g = torch.full((n, 2), -1.0)
    q, k, v = (t.to(DT[dtype]).cuda() for t in (q, k, v))
    o, S = att.gated_linear_attention(q, k, v, g.cuda(), None, None, torch.tensor([0, n], dtype=torch.int32).cuda())
    assert torch.isfinite(o).all() and torch.isfinite(S).all() and S.abs().sum() > 0
