"""Attention over values whose scales lie at the ends of fp32's range, or far
apart, against the 64-bit form: the second product's fp16 operands are held
relative to a power of two for each row, which has to follow the scales without
leaving fp32 itself."""
import pytest
import torch

from mixers_plain import attend, half_step

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture
def att(gpu):
    from breeze_amd import attention
    return attention


def _cache(att, gen, v_scales, D, kind, page=64):
    """One key head's cache in page order: keys of usual size, values of 90 to 120
    (all positive: sums of many do not cancel) times the given scales."""
    n = v_scales.numel()
    P = (n + page - 1) // page
    k = torch.randint(-127, 128, (P, 1, page, D), generator=gen).to(torch.int8)
    v = torch.randint(90, 121, (P, 1, page, D), generator=gen).float()
    if kind == "fp8":
        k, v = (k.float() * 3).to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    else:
        v = v.to(torch.int8)
    ks, vs = torch.full((P, 1, page), 0.01), torch.zeros((P, 1, page))
    vs.view(-1)[:n] = v_scales
    cache = att.KVCache(*(t.cuda() for t in (k, v, ks, vs)))
    return cache, torch.arange(P, dtype=torch.int32)[None]


def _check(got, want, bound, dtype):
    bound = bound + half_step(dtype) * (want.abs() + bound).clamp_min(torch.finfo(dtype).smallest_normal)
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / bound).max().item()
    print(f"error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0


def _run(att, seed, v_scales, kind, dtype, heads, D, q_lens, small=0.0):
    """Sequences that all read the same pages, each ending at the last key; the first
    16 are looked at."""
    gen = torch.Generator().manual_seed(seed)
    cache, table = _cache(att, gen, v_scales, D, kind)
    n, B = v_scales.numel(), len(q_lens)
    q = (0.3 * torch.randn((sum(q_lens), heads, D), generator=gen)).to(DT[dtype])
    table = table.expand(B, -1)
    cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.full((B,), n, dtype=torch.int32).cuda(), cu.cuda())
    q_lens = q_lens[:16]
    T = sum(q_lens)
    want, bound = attend(q[:T], cache, table, [n] * B, q_lens, D ** -0.5, dtype == "fp32")
    _check(got[:T], want, bound + small, DT[dtype])


# Which kernel: 600 single tokens leave one split a sequence; 40 tokens of 4 heads
# are 160 rows; 200 are 800 rows, whose keys are unpacked first.
SHAPES = {"keys": [1] * 600, "rows": [40], "tiles": [200]}


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(SHAPES))
def test_scales_that_fall_by_the_whole_range(att, kind, dtype, D, form):
    """Values of usual size, then some 2^100 smaller, then the smallest: the sums
    of the first may not be multiplied by what the last would like."""
    vs = torch.cat([torch.ones(128), torch.full((128,), 2.0 ** -100), torch.full((128,), 2.0 ** -126)])
    _run(att, 1, vs, kind, dtype, 4, D, SHAPES[form])
    _run(att, 2, vs.flip(0), kind, dtype, 4, D, SHAPES[form])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(SHAPES))
def test_scales_at_the_ends_of_the_range(att, kind, dtype, D, form):
    """All values tiny, or all huge.  A weight errs by no less than 2^-25 in units in
    which a probability of 1 is 2^9 / nu times the value's scale: nu is 2^-110 at
    least, so with scales of 2^-120 each key adds up to 2^-25 * 2^-110 * 2^-9 * 448."""
    n = 300
    _run(att, 3, torch.full((n,), 2.0 ** -120), kind, dtype, 4, D, SHAPES[form], n * 2.0 ** (-25 - 110 - 9) * 448)
    _run(att, 4, torch.full((n,), 2.0 ** 90), kind, dtype, 4, D, SHAPES[form])


@pytest.mark.parametrize("dtype", list(DT))
def test_many_keys_before_a_fall(att, dtype):
    """8192 keys of equal weight and scale 1, then 64 of scale 1e-31, in one prompt
    whose rows are not split: the mean over all keys, where the sums times 2^100
    would be past fp32.  Queries of zeros: o_i is the mean of v_0 .. v_i, in fp16's
    probabilities of one power of two each (exact), so fp32 sums are all that errs:
    i + 1 terms, 2^-24 each."""
    D, heads, n = 64, 8, 8256
    vs = torch.ones(n)
    vs[8192:] = 1e-31
    cache, table = _cache(att, torch.Generator().manual_seed(5), vs, D, "int8")
    cache.v.fill_(100)
    q = torch.zeros((n, heads, D), dtype=DT[dtype], device="cuda")
    lens, cu = torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    got = att.paged_attention(q, cache, table.cuda(), lens, cu).cpu().double()
    want = (100 * vs.double()).cumsum(0) / torch.arange(1, n + 1).double()
    bound = want * (n * 2.0 ** -24 + half_step(DT[dtype]))
    assert torch.isfinite(got).all()
    assert ((got - want[:, None, None]).abs() <= bound[:, None, None]).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_new_largest_score_leaves_small_values_alone(att, kind, dtype):
    """Huge values of small scores, then tiny ones of scores so much larger that the
    former have no weight left: the tiny ones come out, in full precision."""
    for form, q_lens in SHAPES.items():
        for D in (64, 128, 256):
            gen = torch.Generator().manual_seed(6)
            n = 400
            vs = torch.ones(n)
            vs[128:] = 2.0 ** -90
            cache, table = _cache(att, gen, vs, D, kind)
            # Scores of -200 or less for the first 128 keys (whole tiles) against the rest's.
            cache.k.view(torch.int8).fill_(0)
            one = torch.tensor([1.0]).to(cache.k.dtype).view(torch.int8).item()
            cache.k.view(torch.int8).view(-1, D)[:128, 0] = one
            cache.k_scale.fill_(1.0)
            B = len(q_lens)
            q = torch.zeros((sum(q_lens), 4, D))
            q[:, :, 0] = -200 * D ** 0.5
            q = q.to(DT[dtype])
            cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32)
            table = table.expand(B, -1)
            got = att.paged_attention(q.cuda(), cache, table.cuda(), torch.full((B,), n, dtype=torch.int32).cuda(), cu.cuda())
            some = q_lens[:16]
            want, _ = attend(q[:sum(some)], cache, table, [n] * B, some, D ** -0.5, False)
            # Weights of the first keys: exp(-200) = 2^-288 times 120, against 90 * 2^-90: none.
            # The others are equal: their sums err by n 2^-24, their probabilities by fp16's rounding.
            rel = n * 2.0 ** -24 + (2.0 ** -21 if dtype == "fp32" else half_step(torch.float16)) + half_step(DT[dtype])
            assert ((got[:sum(some)].cpu().double() - want).abs() <= 2 * rel * want.abs()).all(), (form, D)
