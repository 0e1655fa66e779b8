"""Attention of trees over values whose scales lie at the ends of fp32's range, or
far apart: as causal attention's tests of them, with chains, whose nodes see what
causal tokens see."""
import pytest
import torch

from drafts_plain import cu_of
from mixers_plain import attend, half_step
from test_gpu_attn_value_scales import DT, _cache, _check

pytestmark = pytest.mark.gpu

# One node of 600 sequences, chains of up to 32, 64 and 128 rows a key head, and one that is cut into several units.
SHAPES = {"ones": [1] * 600, "few": [8] * 20, "some": [16], "many": [32] * 3, "long": [100]}


@pytest.fixture
def mods(gpu):
    from breeze_amd import attention, drafts
    return attention, drafts


def _run(mods, seed, v_scales, kind, dtype, D, q_lens, small=0.0):
    att, drafts = mods
    gen = torch.Generator().manual_seed(seed)
    cache, table = _cache(att, gen, v_scales, D, kind)
    n, B, heads = v_scales.numel(), len(q_lens), 4
    q = (0.3 * torch.randn((sum(q_lens), heads, D), generator=gen)).to(DT[dtype])
    table = table.expand(B, -1)
    parents = torch.cat([torch.arange(-1, k - 1) for k in q_lens]).to(torch.int32)
    got = drafts.tree_attention(q.cuda(), cache, table.cuda(), torch.full((B,), n, dtype=torch.int32).cuda(),
                                parents.cuda(), cu_of(q_lens).cuda())
    q_lens = q_lens[:16]
    T = sum(q_lens)
    want, bound = attend(q[:T], cache, table, [n] * B, q_lens, D ** -0.5, dtype != "bf16")
    _check(got[:T], want, bound + small, DT[dtype])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(SHAPES))
def test_scales_that_fall_by_the_whole_range(mods, kind, dtype, D, form):
    """A fp16 output's own range ends at 2^16: values of usual size there."""
    vs = torch.cat([torch.ones(128), torch.full((128,), 2.0 ** -100), torch.full((128,), 2.0 ** -126)])
    _run(mods, 1, vs, kind, dtype, D, SHAPES[form])
    _run(mods, 2, vs.flip(0), kind, dtype, D, SHAPES[form])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(SHAPES))
def test_scales_at_the_ends_of_the_range(mods, kind, dtype, D, form):
    """All values tiny, or all huge.  A weight errs by no less than 2^-25 in units in
    which a probability of 1 is 2^9 / nu times the value's scale: nu is 2^-110 at
    least, so with scales of 2^-120 each key adds up to 2^-25 * 2^-110 * 2^-9 * 448."""
    n = 300
    _run(mods, 3, torch.full((n,), 2.0 ** -120), kind, dtype, D, SHAPES[form], n * 2.0 ** (-25 - 110 - 9) * 448)
    _run(mods, 4, torch.full((n,), 2.0 ** 90), kind, dtype, D, SHAPES[form])
