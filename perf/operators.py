"""The decoder's token mixers, as timed cases: what runs between the quantized
projections of a layer.

Each case is one call (or one pair of calls) of ``breeze_amd.attention`` on GPU
tensors:

- ``kv``: the keys and values of new tokens quantized into the pages of a
  cache, and the same tokens read back from it;
- ``attn``: attention of new tokens (one a sequence, or a chunk) over that
  cache, causal among the new tokens;
- ``gla``: gated linear attention, with the delta rule where ``beta`` is true:
  one token a sequence from a kept state, or whole prompts.

``q_lens`` and ``ctx`` give the new tokens and the cached tokens in front of
them for each sequence: ``"5,1,77"`` one by one, ``"64x1"`` that many alike,
``"64x1-8000"`` that many spread over the logarithm (with ``spread``, the seed
of that spread).  ``kind`` is what the cache holds: INT8 with one fp32 scale
for each token and head, or e4m3 with a power of two for each.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_KV = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


_module = None


def _attention():
    global _module
    if _module is not None:
        return _module
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "breeze-engine_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from breeze_amd import attention

    _module = attention
    return attention


# ------------------------------------------------------------------ cases

def _kv(tokens, heads, dim, page, kind, dtype):
    return dict(op="kv", tokens=tokens, kv_heads=heads, dim=dim, page=page, kind=kind, dtype=dtype)


def _attn(q_lens, ctx, heads, kv_heads, dim, page, kind, dtype, spread=0):
    return dict(op="attn", q_lens=q_lens, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind,
                dtype=dtype, spread=spread)


def _gla(q_lens, k_heads, v_heads, dim, beta, dtype, spread=0):
    return dict(op="gla", q_lens=q_lens, k_heads=k_heads, v_heads=v_heads, dim=dim, beta=beta, dtype=dtype,
                spread=spread)


def listed():
    return [
        # One decode step's token, the full-attention layers' heads of the 27B
        # decoder (k and v projections of 1024 columns): latency.
        dict(_kv(1, 4, 256, 16, "int8", "fp32"), name="kv_one"),
        # A prompt's keys and values at once.
        dict(_kv(8192, 4, 256, 64, "int8", "fp32"), name="kv_prompt"),
        # An odd number of tokens, e4m3, smaller heads and pages.
        dict(_kv(4999, 8, 128, 16, "fp8", "bf16"), name="kv_fp8_ragged"),
        # Single-token decode of one sequence.
        dict(_attn("1", "4100", 24, 4, 256, 16, "int8", "fp32"), name="attn_one"),
        # A serving batch's decode step: 64 sequences of very different lengths.
        dict(_attn("64x1", "64x100-16000", 32, 8, 128, 16, "fp8", "bf16", spread=3), name="attn_batch"),
        # A chunk of a long prompt, most of which is cached already.
        dict(_attn("1024", "31744", 24, 4, 256, 64, "int8", "fp32"), name="attn_chunk_long"),
        # Mixed batch: short prompts, chunks of odd lengths, single tokens.
        dict(_attn("1,700,33,1,257,5,1,129", "5000,0,64,1023,4097,17,0,2500", 32, 8, 128, 32, "int8", "bf16"),
             name="attn_mixed"),
        # A whole prompt with nothing cached before it.
        dict(_attn("4096", "0", 32, 8, 128, 64, "fp8", "fp16"), name="attn_prompt"),
        # Single-token decode of one sequence, the linear-attention layers' heads
        # of the 27B decoder (16 key heads, 48 value heads of 128).
        dict(_gla("1", 16, 48, 128, True, "fp32"), name="gla_one"),
        # A serving batch's decode step.
        dict(_gla("64x1", 16, 48, 128, True, "bf16"), name="gla_batch"),
        # A prompt of one sequence.
        dict(_gla("4096", 16, 48, 128, True, "fp32"), name="gla_prompt"),
        # Short prompts of ragged lengths, decay without the delta rule.
        dict(_gla("300,1,1000,77,64,513", 32, 32, 128, False, "bf16"), name="gla_ragged"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "gla"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "kv":
        heads, dim = rng.choice([(4, 256), (8, 128), (2, 64), (1, 128)])
        return _kv(_log(rng, 1, 8192), heads, dim, rng.choice([16, 32, 64, 128]), rng.choice(["int8", "fp8"]), dtype)
    if op == "attn":
        heads, kv_heads, dim = rng.choice([(24, 4, 256), (32, 8, 128), (16, 2, 64), (8, 8, 128)])
        page, kind = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "fp8"])
        if rng.random() < 0.5:  # single tokens
            n = _log(rng, 1, 64)
            hi = _log(rng, 64, 16000)
            return _attn("%dx1" % n, "%dx1-%d" % (n, hi), heads, kv_heads, dim, page, kind, dtype, rng.randrange(1 << 20))
        n = rng.choice([1, 1, 2, 3, 5])
        hi_q, hi_c = _log(rng, 2, 2048 // n), _log(rng, 1, 16000)
        return _attn("%dx1-%d" % (n, hi_q), "%dx1-%d" % (n, hi_c), heads, kv_heads, dim, page, kind, dtype,
                     rng.randrange(1 << 20))
    k_heads, v_heads, dim = rng.choice([(16, 48, 128), (16, 32, 128), (8, 8, 64), (32, 32, 128)])
    beta = rng.random() < 0.7
    if rng.random() < 0.5:
        return _gla("%dx1" % _log(rng, 1, 64), k_heads, v_heads, dim, beta, dtype)
    n = rng.choice([1, 1, 2, 4, 7])
    return _gla("%dx1-%d" % (n, _log(rng, 2, 2048)), k_heads, v_heads, dim, beta, dtype, rng.randrange(1 << 20))


def _lens(text, rng):
    if "x" not in text:
        return [int(t) for t in text.split(",")]
    n, of = text.split("x")
    if "-" not in of:
        return [int(of)] * int(n)
    lo, hi = (int(t) for t in of.split("-"))
    return [_log(rng, lo, hi) for _ in range(int(n))]


def _shape(case):
    """New tokens and cached tokens of each sequence."""
    rng = random.Random(case["spread"])
    q = _lens(case["q_lens"], rng)
    return q, (_lens(case["ctx"], rng) if "ctx" in case else [0] * len(q))


# ------------------------------------------------------------------ inputs

class _State:
    pass


def _quantized(x, kind):
    """Cache values and scales of fp32 rows [..., D]."""
    top = x.abs().amax(-1)
    if kind == "int8":
        scale = (top.double() / 127).float()
        y = x.double() / torch.where(scale > 0, scale, 1.0).double().unsqueeze(-1)
        return y.round().clamp(-127, 127).to(torch.int8), scale
    # The smallest power of two that brings the row within 448 (1.75 * 2^8).
    man, exp = torch.frexp(top)
    e = torch.where(man > 0.875, exp - 8, exp - 9).clamp_min(-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), 0.0)
    y = x / torch.where(scale > 0, scale, 1.0).unsqueeze(-1)
    return y.to(torch.float8_e4m3fn), scale


def _values(gen, *shape):
    """Keys or values: channels of unlike size, as projections give them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return x * torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device="cuda"))


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    s = _State()
    s.case = case
    s.handle = None  # the cache object, which a program makes once
    dtype = _DT[case["dtype"]]
    dev = "cuda"
    if case["op"] == "gla":
        lens, _ = _shape(case)
        s.lens, T, D = lens, sum(lens), case["dim"]
        Hk, Hv = case["k_heads"], case["v_heads"]
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        # One projection's columns, as the layer's input projection gives them.
        qkv = torch.empty((T, (2 * Hk + Hv) * D), dtype=dtype, device=dev)
        s.q, s.k, s.v = (x.view(T, -1, D) for x in qkv.split([Hk * D, Hk * D, Hv * D], dim=1))
        s.q.copy_(unit(torch.randn((T, Hk, D), generator=gen, device=dev)))
        s.k.copy_(unit(torch.randn((T, Hk, D), generator=gen, device=dev)))
        s.v.copy_(torch.randn((T, Hv, D), generator=gen, device=dev))
        # Decays from nearly none to a fast one, as softplus(dt) * A gives them.
        A = torch.exp(torch.rand((Hv,), generator=gen, device=dev) * math.log(16))
        dt = torch.exp(torch.rand((T, Hv), generator=gen, device=dev) * 4.6 - 6.9)
        s.g = -A * dt
        s.beta = torch.sigmoid(torch.randn((T, Hv), generator=gen, device=dev)) if case["beta"] else None
        s.state = 0.3 * torch.randn((len(lens), Hv, D, D), generator=gen, device=dev)
        s.cu = _cu(lens)
        s.single = max(lens) == 1
        return s
    H, D, page, kind = case["kv_heads"], case["dim"], case["page"], case["kind"]
    if case["op"] == "kv":
        T = case["tokens"]
        s.k, s.v = (_values(gen, T, H, D).to(dtype) for _ in range(2))
        pages = (T + page - 1) // page + 3
        order = torch.randperm(pages, generator=gen, device=dev)
        # A prompt fills its pages in order; the pages are anywhere.
        at = torch.arange(T, device=dev)
        s.slots = (order[at // page] * page + at % page).to(torch.int32)
        s.cache = [torch.zeros((pages, H, page, D), dtype=torch.int8, device=dev).view(_KV[kind]) for _ in range(2)]
        s.cache += [torch.zeros((pages, H, page), dtype=torch.float32, device=dev) for _ in range(2)]
        return s
    q_lens, ctx = _shape(case)
    s.q_lens, s.kv = q_lens, [c + n for c, n in zip(ctx, q_lens)]
    need = [(n + page - 1) // page for n in s.kv]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    s.table = torch.zeros((len(need), max(need)), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        s.table[b, :n] = order[at:at + n]
        at += n
    s.cache = [torch.empty((pages, H, page, D), dtype=torch.int8, device=dev).view(_KV[kind]) for _ in range(2)]
    s.cache += [torch.empty((pages, H, page), dtype=torch.float32, device=dev) for _ in range(2)]
    for i in range(2):
        bias = torch.exp(0.5 * torch.randn((H, 1, D), generator=gen, device=dev))
        for p in range(0, pages, 4096):
            part = torch.randn((min(4096, pages - p), H, page, D), generator=gen, device=dev) * bias
            y, sc = _quantized(part, kind)
            s.cache[i][p:p + 4096].view(torch.int8).copy_(y.view(torch.int8))
            s.cache[2 + i][p:p + 4096] = sc
    T = sum(q_lens)
    s.q = (1.5 * torch.randn((T, case["heads"], D), generator=gen, device=dev)).to(dtype)
    s.kv_lens = torch.tensor(s.kv, dtype=torch.int32, device=dev)
    s.cu = _cu(q_lens)
    s.single = max(q_lens) == 1
    return s


# ------------------------------------------------------------------ one pass

def _run_own(s):
    a = _attention()
    c = s.case
    if c["op"] == "gla":
        return a.gated_linear_attention(s.q, s.k, s.v, s.g, s.beta, s.state, None if s.single else s.cu)
    if s.handle is None:
        s.handle = a.KVCache(*s.cache)
    cache = s.handle
    if c["op"] == "kv":
        a.kv_write(cache, s.k, s.v, s.slots)
        return a.kv_read(cache, s.slots, s.k.dtype)
    return a.paged_attention(s.q, cache, s.table, s.kv_lens, None if s.single else s.cu)


def _run_kv(s):
    c = s.case
    page = c["page"]
    slots = s.slots.long()
    out = []
    for i, x in enumerate((s.k, s.v)):
        y, scale = _quantized(x.float(), c["kind"])
        at = (slots // page, slice(None), slots % page)
        s.cache[i].view(torch.int8)[at] = y.view(torch.int8)
        s.cache[2 + i][at] = scale
        back = s.cache[i].view(torch.int8)[at].view(_KV[c["kind"]]).float() * s.cache[2 + i][at].unsqueeze(-1)
        out.append(back.to(x.dtype))
    return tuple(out)


def _padded(cu, n):
    """Row numbers of the packed tokens, [sequences, n], and which are real."""
    at = cu[:-1, None].long() + torch.arange(n, device=cu.device)
    real = at < cu[1:, None]
    return torch.where(real, at, 0), real


def _run_attn(s):
    c = s.case
    page, Hq, H, D = c["page"], c["heads"], c["kv_heads"], c["dim"]
    B, G, n, keys = len(s.kv), c["heads"] // c["kv_heads"], max(s.q_lens), max(s.kv)
    at, real = _padded(s.cu, n)
    q = s.q.float()[at].view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    j = torch.arange(keys, device="cuda")
    where = (s.table.long()[:, j // page], slice(None), j % page)

    def gathered(i):  # [B, H, keys, D]
        x = s.cache[i].view(torch.int8)[where].view(_KV[c["kind"]]).float() * s.cache[2 + i][where].unsqueeze(-1)
        return x.permute(0, 2, 1, 3)

    scores = torch.matmul(q, gathered(0).transpose(2, 3).contiguous()).view(B, H, G, n, keys) / math.sqrt(D)
    # New token i of a sequence sees its cached tokens and the new ones up to itself.
    q_len = (s.cu[1:] - s.cu[:-1])[:, None, None]
    last = (s.kv_lens[:, None, None] - q_len) + torch.arange(n, device="cuda")[None, :, None]
    seen = (j <= last) & real[:, :, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, H, G * n, keys), gathered(1).contiguous()).view(B, H, G, n, D)
    out = out / total.clamp_min(1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[real].to(s.q.dtype)


def _run_gla(s):
    c = s.case
    D, rep, n = c["dim"], c["v_heads"] // c["k_heads"], max(s.lens)
    at, real = _padded(s.cu, n)
    wide = lambda x: x.float()[at].repeat_interleave(rep, dim=2)  # noqa: E731
    q, k, v = wide(s.q) / math.sqrt(D), wide(s.k), s.v.float()[at]
    # Past a sequence's end nothing decays and nothing is added.
    keep = torch.where(real[:, :, None], torch.exp(s.g)[at], 1.0)
    k = k * real[:, :, None, None]
    beta = None if s.beta is None else s.beta[at].unsqueeze(-1)
    state, out = s.state.clone(), torch.empty_like(v)
    # The recurrence itself: each token needs the state that the one before it left.
    for t in range(n):
        state *= keep[:, t, :, None, None]
        u = v[:, t]
        if beta is not None:
            u = beta[:, t] * (u - (state * k[:, t].unsqueeze(-1)).sum(-2))
        state += k[:, t].unsqueeze(-1) * u.unsqueeze(-2)
        out[:, t] = (state * q[:, t].unsqueeze(-1)).sum(-2)
    return out[real].to(s.q.dtype), state


def run(s):
    if own:
        return _run_own(s)
    return {"kv": _run_kv, "attn": _run_attn, "gla": _run_gla}[s.case["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "kv":
        rows = 2 * case["tokens"] * case["kv_heads"]
        D = case["dim"]
        # New values in, cache values and scales out and back in, values out; slots twice.
        return {"bytes": rows * (2 * D * e + 2 * (D + 4)) + 8 * case["tokens"], "flops": 3 * rows * D}
    q, ctx = _shape(case)
    T, D = sum(q), case["dim"]
    if case["op"] == "attn":
        kv = sum(q) + sum(ctx)
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(q, ctx))
        b = 2 * T * case["heads"] * D * e + 2 * kv * case["kv_heads"] * (D + 4) + 4 * kv // case["page"]
        return {"bytes": b, "flops": 4 * D * case["heads"] * pairs}
    Hk, Hv = case["k_heads"], case["v_heads"]
    b = T * (2 * Hk + 2 * Hv) * D * e + T * Hv * (8 if case["beta"] else 4) + 8 * len(q) * Hv * D * D
    return {"bytes": b, "flops": T * Hv * D * D * (6 if case["beta"] else 4)}


# ------------------------------------------------------------------ in 64 bits

def _exact_row_values(x, kind):
    """What the cache holds for fp64 rows [..., D], as the values it stands for."""
    top = x.abs().amax(-1, keepdim=True)
    if kind == "int8":
        scale = (top / 127).float().double()  # a scale is an fp32 number
        return torch.where(scale > 0, (x / scale).round().clamp(-127, 127) * scale, 0.0)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp_min(1e-300) / 448)).clamp_min(-126))
    y = x / scale
    # e4m3: 4 significant bits, and steps of 2^-9 below 2^-6.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / step).round() * step * scale


def _exact_attn(s, c):
    H, G, page, D = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"], c["dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, keys) in enumerate(zip(s.q_lens, s.kv)):
        pages = s.table[b, :(keys + page - 1) // page].long()
        for h in range(H):
            k, v = (s.cache[i].view(torch.int8)[pages, h].view(_KV[c["kind"]]).double().reshape(-1, D)[:keys]
                    * s.cache[2 + i][pages, h].double().reshape(-1, 1)[:keys] for i in range(2))
            hidden = torch.arange(keys, device="cuda")[None] > torch.arange(keys - n, keys, device="cuda")[:, None]
            for g in range(h * G, h * G + G):
                x = s.q[start:start + n, g].double() @ k.t() * D ** -0.5
                p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
                out[start:start + n, g] = p @ v
        start += n
    return out


def _exact_gla(s, c):
    rep = c["v_heads"] // c["k_heads"]
    outs, states, start = [], [], 0
    for b, n in enumerate(s.lens):
        part = slice(start, start + n)
        q, k = (x[part].double().repeat_interleave(rep, dim=1) for x in (s.q, s.k))
        v, a = s.v[part].double(), s.g[part].double().exp()
        S = s.state[b].double()
        o = torch.empty_like(v)
        for t in range(n):
            S = S * a[t][:, None, None]
            u = v[t]
            if s.beta is not None:
                u = (u - torch.bmm(k[t][:, None], S)[:, 0]) * s.beta[part][t].double()[:, None]
            S = torch.baddbmm(S, k[t][:, :, None], u[:, None])
            o[t] = torch.bmm(q[t][:, None], S)[:, 0]
        outs.append(o * c["dim"] ** -0.5)
        states.append(S)
        start += n
    return torch.cat(outs), torch.stack(states)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "kv":
        return tuple(_exact_row_values(x.double(), case["kind"]) for x in (s.k, s.v))
    return _exact_attn(s, case) if case["op"] == "attn" else _exact_gla(s, case)
