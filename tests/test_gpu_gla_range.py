"""Gated linear attention of prompts: what their products keep, states far larger
than what is added to them, and long prompts, which go in segments."""
import pytest
import torch

from breeze_amd import hip_backend as hb
from mixers_plain import recur

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [100, 300, 700])
def test_a_large_state_and_tiny_additions(att, delta, n):
    """A state of 1e10 to which products of 1e-38 are added, chunk after chunk: it
    stays, within its fp32 products' errors, and does not leave fp32 in the units
    of what is added."""
    gen = torch.Generator().manual_seed(n)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    Hv, Dk, Dv = 2, 64, 48
    q, k, v = rand(n, 1, Dk), 1e-19 * rand(n, 1, Dk), 1e-19 * rand(n, Hv, Dv)
    g, state = torch.full((n, Hv), -1e-3), 1e10 * rand(1, Hv, Dk, Dv)
    beta = torch.sigmoid(rand(n, Hv)) if delta else None
    o, S = att.gated_linear_attention(*(None if t is None else t.cuda() for t in (q, k, v, g, beta, state)), _cu([n]).cuda())
    want_o, want_S, _ = recur(q, k, v, g, beta, state, [n], Dk ** -0.5)
    # A chunk multiplies the state by one decay (an exponential's last bits and one
    # rounding, 2^-22) and rounds it; rows of O have 64 terms of 22 bits and the like.
    chunks = -(-n // 64)
    assert torch.isfinite(S).all() and torch.isfinite(o).all()
    assert ((S.cpu().double() - want_S).abs() <= (chunks + 1) * 2.0 ** -22 * state.double().abs()).all()
    size = (q.double().abs().repeat(1, Hv, 1).unsqueeze(-1) * state[0].double().abs()).sum(2) * Dk ** -0.5
    assert ((o.cpu().double() - want_o).abs() <= (chunks + 66) * 2.0 ** -21 * size).all()


def _excess_norm(got, want):
    """The norm of what is left of |got - want| after one rounding to got's type."""
    f = torch.finfo(got.dtype)
    got, off = got.double(), (got.double() - want).abs()
    step = torch.exp2(torch.floor(torch.log2(torch.maximum(got.abs(), want.abs()).clamp_min(f.smallest_normal)))) * f.eps
    return (off - step / 2).clamp_min(0).norm()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(2, 6, 128, 128), (1, 2, 64, 80)])
@pytest.mark.parametrize("lens", [[64], [130, 17, 300], [700]])
def test_fp16_rows_are_rounded_once(att, delta, Hk, Hv, Dk, Dv, lens):
    """Rows of fp16 prompts: products of 22 bits, then one rounding.  |o - want| is at
    most half a step plus the error before it; the latter's norm is at most 5 sqrt(c)
    2^-20 of the rows' and state's (five products in a row, c chunks), so what is left
    over half a step has no larger one.  Operands of 11 bits would leave 2^-13."""
    gen = torch.Generator().manual_seed(len(lens))
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    T = sum(lens)
    q, k, v = unit(rand(T, Hk, Dk)).half(), (0.999 * unit(rand(T, Hk, Dk))).half(), rand(T, Hv, Dv).half()
    g, state = -torch.exp(3 * torch.rand((T, Hv), generator=gen) - 4), rand(len(lens), Hv, Dk, Dv)
    beta = torch.sigmoid(rand(T, Hv)) if delta else None
    o, _ = att.gated_linear_attention(*(None if t is None else t.cuda() for t in (q, k, v, g, beta, state)), _cu(lens).cuda())
    want, _, size = recur(q, k, v, g, beta, state, lens, Dk ** -0.5)
    start = 0
    for b, n in enumerate(lens):
        part = slice(start, start + n)
        rel = 5 * (-(-n // 64)) ** 0.5 * 2.0 ** -20
        whole = want[part].norm() + Dk ** -0.5 * size[b].norm() * q[part].double().norm(dim=-1).max()
        left = _excess_norm(o[part].cpu(), want[part])
        print(f"{n} tokens: {(left / (rel * whole)).item():.3f} of the bound", flush=True)
        assert left <= rel * whole
        start += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[9000, 5, 0, 31500, 70, 12345], [31000, 31000], [45000]])
def test_long_prompts_in_segments(att, dtype, lens):
    """More chunks than the workspace holds at once (about 30000 tokens of these heads in
    fp32, 38000 in bf16), in one call and sequence by sequence, long ones in parts:
    the same bits, since a state's units are powers of two."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    Hk, Hv, D, T = 16, 48, 128, sum(lens)
    assert hb._lib.i4_gated_linear_attention_workspace(T, len(lens), Hk, Hv, D, D, 0 if dtype == torch.float32 else 1, 1, 1) > 0.99 * 2 ** 30
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k, v = unit(rand(T, Hk, D)).to(dtype), unit(rand(T, Hk, D)).to(dtype), rand(T, Hv, D).to(dtype)
    g, beta = -torch.exp(-7 + 5 * torch.rand((T, Hv), generator=gen, device="cuda")), torch.sigmoid(rand(T, Hv))
    state = rand(len(lens), Hv, D, D)
    want = state.clone()
    o, S = att.gated_linear_attention(q, k, v, g, beta, state, _cu(lens).cuda())
    o2, S2 = att.gated_linear_attention(q, k, v, g, beta, want.clone(), _cu(lens).cuda())  # the workspace holds the last call's
    assert torch.equal(o, o2) and torch.equal(S, S2) and torch.equal(state, want)
    start = 0
    for b, n in enumerate(lens):
        s, at = want[b:b + 1].clone(), start
        while at < start + n or n == 0:
            part = min(230 * 64, start + n - at)  # whole chunks, but for the last
            cut = slice(at, at + part)
            x, _ = att.gated_linear_attention(q[cut], k[cut], v[cut], g[cut], beta[cut], s, _cu([part]).cuda(), state_out=s)
            assert torch.equal(x, o[cut]), (b, at)
            at += part
            if n == 0:
                break
        assert torch.equal(s[0], S[b]), b
        start += n
    # In place, and from zeros.
    att.gated_linear_attention(q, k, v, g, beta, state, _cu(lens).cuda(), state_out=state)
    assert torch.equal(state, S)
    a = att.gated_linear_attention(q, k, v, g, beta, None, _cu(lens).cuda())
    b = att.gated_linear_attention(q, k, v, g, beta, torch.zeros_like(state), _cu(lens).cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
