"""Plain 64-bit forms of the token mixers, for their tests."""
import numpy as np
import torch

F64 = torch.float64


def half_step(dtype):
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def quantize(x, kind):
    """fp64 rows [..., D] -> (stored numbers as fp64, scales as fp64)."""
    top = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    if kind == "int8":
        s = (top / 127).float().double()
        y = torch.where(s > 0, x / torch.where(s > 0, s, 1.0), 0.0).round().clamp(-127, 127)
    else:
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448)).clamp_min(-126)
        s = torch.where(top > 0, torch.exp2(e), 0.0)
        y = torch.where(s > 0, x / torch.where(s > 0, s, 1.0), 0.0)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        y = (y / step).round() * step
    return torch.where(bad, 0.0, y), torch.where(bad, torch.nan, s).squeeze(-1)


def page_values(pages):
    """Stored numbers of a page tensor as fp64."""
    if pages.dtype == torch.int8:
        return pages.cpu().double()
    b = pages.view(torch.int8).cpu().numpy().view(np.uint8).astype(np.int64)
    sign, e, m = np.where(b & 128, -1.0, 1.0), (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return torch.from_numpy(sign * v)


def sequence_values(pages, scales, table, n, page):
    """fp64 [n, H, D] of the first n keys of a page list; NaN rows become zeros
    that `ok` [n] marks where the page is not the cache's."""
    P, H, _, D = pages.shape
    j = torch.arange(n)
    pg = torch.as_tensor(table, dtype=torch.int64)[j // page] if n else j
    ok = (pg >= 0) & (pg < P)
    pg = torch.where(ok, pg, 0)
    return pages[pg, :, j % page] * scales[pg, :, j % page].unsqueeze(-1), ok


def attend(q, cache, table, kv_lens, q_lens, scale, split):
    """(out, bound): fp64 attention of packed q [T, heads, D] and how far fp32
    sums over fp16 products of the documented precision may be from it."""
    kp, vp = page_values(cache.k), page_values(cache.v)
    ks, vs = cache.k_scale.cpu().double(), cache.v_scale.cpu().double()
    page, H = cache.page_size, cache.kv_heads
    heads, D = q.shape[1:]
    G = heads // H
    q = q.cpu().double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    start = 0
    for b, n in enumerate(q_lens):
        kv = min(max(int(kv_lens[b]), 0), table.shape[1] * page)
        rows = torch.arange(n)
        if kv and n:
            k, ok = sequence_values(kp, ks, table[b], kv, page)
            v, _ = sequence_values(vp, vs, table[b], kv, page)
            seen = (torch.arange(kv)[None] <= (kv - n + rows)[:, None]) & ok[None]  # [n, kv]
            k, v = (torch.where(ok[:, None, None], x, 0.0) for x in (k, v))
            for h in range(heads):
                x, kk, vv = q[start:start + n, h], k[:, h // G], v[:, h // G]
                spoilt = torch.isnan(kk).any(-1) | torch.isnan(vv).any(-1)  # keys whose rows read back as NaN
                kk, vv = kk.nan_to_num(0), vv.nan_to_num(0)
                s = (x @ kk.t()) * scale
                size = (x.abs() @ kk.abs().t()) * scale
                s = torch.where(seen, s, -torch.inf)
                top = s.amax(-1, keepdim=True)
                top = torch.where(torch.isinf(top), 0.0, top)
                p = torch.where(seen, torch.exp(s - top), 0.0)
                l = p.sum(-1, keepdim=True)
                p = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
                o = torch.where((seen & spoilt).any(-1, keepdim=True), torch.nan, p @ vv)
                # Each probability: the score's error (the product's fp32 sums over D
                # terms, the query's 22 bits, three roundings of the scale, exponent
                # and difference), the exponential's two last bits, its own rounding
                # for the product; then the fp32 sums over the keys.
                arg = torch.where(seen, (s - top).abs(), 0.0)
                err = size * (D * 2.0 ** -24 + 2.0 ** -22) + (arg + s.abs().where(seen, torch.zeros(()).double())) * 2.0 ** -22
                err = err + 2.0 ** -22 + (2.0 ** -21 if split else half_step(torch.float16)) + kv * 2.0 ** -24
                pv = p * err
                worst = pv @ vv.abs() + pv.sum(-1, keepdim=True) * (p @ vv.abs())
                # A weight errs by no less than half of fp16's smallest step, 2^-25, in units
                # in which a probability of 1 times the tile's largest value scale is 2^9 / 16
                # or more: 2^-30 of the largest value for each key.
                small = 2.0 ** -30 * seen.sum(-1, keepdim=True) * vv.abs().max()
                out[start:start + n, h], bound[start:start + n, h] = o, worst + small
        start += n
    return out, bound


def recur(q, k, v, g, beta, state, q_lens, scale):
    """(o, state, size) of the gated recurrence in fp64; size [B, Hv, Dv] is the
    largest norm of a state's column, or of a token's v there, on the way."""
    rep = v.shape[1] // k.shape[1]
    q, k = (x.cpu().double().repeat_interleave(rep, 1) for x in (q, k))
    v, g = v.cpu().double(), g.cpu().double()
    Hv, Dk, Dv = v.shape[1], q.shape[2], v.shape[2]
    o = torch.zeros_like(v)
    states, sizes, start = [], [], 0
    for b, n in enumerate(q_lens):
        S = torch.zeros((Hv, Dk, Dv), dtype=F64) if state is None else state[b].cpu().double()
        size = S.norm(dim=1)
        for t in range(start, start + n):
            S = S * g[t].exp()[:, None, None]
            u = v[t]
            if beta is not None:
                u = beta[t].cpu().double()[:, None] * (u - (k[t][:, None] @ S)[:, 0])
            S = S + k[t][:, :, None] * u[:, None]
            o[t] = scale * (q[t][:, None] @ S)[:, 0]
            size = torch.maximum(size, torch.maximum(S.norm(dim=1), v[t].abs() * k[t].norm(dim=1)[:, None]))
        states.append(S)
        sizes.append(size)
        start += n
    return o, torch.stack(states), torch.stack(sizes)
