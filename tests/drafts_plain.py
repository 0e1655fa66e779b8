"""Plain forms of a step with drafted tokens, for its tests: whole numbers in
Python, the rest in 64 bits."""
import math

import torch

from mixers_plain import half_step, page_values, sequence_values

NODES = 1024  # of a tree


def tree(n, gen, chain=False, roots=1):
    """Parents of a random tree of n nodes, parents first."""
    out = []
    for i in range(n):
        if i < roots:
            out.append(-1)
        elif chain:
            out.append(i - 1)
        else:
            out.append(int(torch.randint(max(0, (i - 1) // 4), i, (1,), generator=gen)))
    return out


def ancestors(parents, i):
    """Node i and what lies above it."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def attend_tree(q, cache, table, kv_lens, trees, scale, split):
    """(out, bound): fp64 attention of packed q [T, heads, D] over each tree's context,
    its ancestors and itself, and how far fp32 sums over fp16 products of the
    documented precision may be from it."""
    kp, vp = page_values(cache.k), page_values(cache.v)
    ks, vs = cache.k_scale.cpu().double(), cache.v_scale.cpu().double()
    page, H = cache.page_size, cache.kv_heads
    heads, D = q.shape[1:]
    G = heads // H
    q = q.cpu().double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    start = 0
    for b, parents in enumerate(trees):
        n = len(parents)
        kv = min(max(int(kv_lens[b]), 0), table.shape[1] * page)
        if n > NODES:
            out[start:start + n] = torch.nan
        elif kv and n:
            k, ok = sequence_values(kp, ks, table[b], kv, page)
            v, _ = sequence_values(vp, vs, table[b], kv, page)
            seen = torch.zeros((n, kv), dtype=torch.bool)
            ctx = kv - n
            seen[:, :max(ctx, 0)] = True
            for i in range(n):
                for j in ancestors(parents, i):
                    if ctx + j >= 0:
                        seen[i, ctx + j] = True
            seen &= ok[None]
            k, v = (torch.where(ok[:, None, None], x, 0.0) for x in (k, v))
            for h in range(heads):
                x, kk, vv = q[start:start + n, h], k[:, h // G], v[:, h // G]
                spoilt = torch.isnan(kk).any(-1) | torch.isnan(vv).any(-1)
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
                err = size * (D * 2.0 ** -24 + 2.0 ** -22)
                err = err + (arg + torch.where(seen, s.abs(), 0.0)) * 2.0 ** -22
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


class Pages:
    """A page table in Python lists."""

    def __init__(self, table, held, free, page):
        self.table, self.held, self.free, self.page = [list(r) for r in table], list(held), list(free), page

    def extend(self, lens, new, parents=None):
        """(slots, positions, kv_lens); parents: a list for each sequence."""
        slots, positions, kv = [], [], []
        out_of_pages = False
        for b, (n, m) in enumerate(zip(lens, new)):
            row, cols = self.table[b], len(self.table[b])
            want = -(-(n + m) // self.page)
            fits = n >= 0 and want <= cols and not (parents and m > NODES)
            need = max(want - self.held[b], 0) if fits else 0
            if need and (out_of_pages or need > len(self.free)):
                out_of_pages, fits = True, False
            if fits:
                for _ in range(need):
                    row[self.held[b]] = self.free.pop()
                    self.held[b] += 1
            for i in range(m):
                at = n + i
                slots.append(row[at // self.page] * self.page + at % self.page if fits else -1)
                deep = len(ancestors(parents[b], i)) - 1 if parents and m <= NODES else i
                positions.append(n + deep)
            kv.append(n + m if fits else -1)
        return slots, positions, kv

    def trim(self, lens):
        gone = []
        for b, n in enumerate(lens):
            keep = self.held[b] if n < 0 else min(self.held[b], -(-n // self.page))
            for j in range(keep, self.held[b]):
                gone.append(self.table[b][j])
                self.table[b][j] = -1
            self.held[b] = keep
        self.free += gone[::-1]


def walk(logits, tokens, parents, uniforms, temperature, draft=None):
    """One sequence's (new tokens, path) by the rule as it is told: a residual
    distribution for each rejected child.  fp64 rows on the CPU."""
    n, V = logits.shape
    node, path, got = 0, [0], []
    u = uniforms.double().tolist()
    while True:
        l = logits[node].double()
        good = bool((l < math.inf).all()) and bool((l > -math.inf).any())
        if not good or not 0 <= temperature < math.inf:
            return got + [-1], path
        if temperature == 0:
            r = torch.zeros_like(l)
            r[int((l == l.max()).nonzero()[0])] = 1.0
        else:
            r = torch.exp((l - l.max()) / temperature)
            r = r / r.sum()
        q = None if draft is None else draft[node].double().clone()
        left, down, gone = 1.0, -1, set()
        for i in range(node + 1, n):
            if parents[i] != node:
                continue
            x = int(tokens[i])
            if not 0 <= x < V or x in gone or not left > 0:
                continue
            if temperature == 0:
                if r[x] == 1:
                    down = i
                    break
                continue
            if u[i] * (1.0 if q is None else float(q[x]) / left) < float(r[x]):
                down = i
                break
            rest = r.clone() if q is None else torch.clamp(r - q / left, min=0.0)
            if q is not None:
                left -= float(q[x])
                q[x] = 0.0
            gone.add(x)
            rest[x] = 0.0
            r = rest / rest.sum()
        if down < 0:
            break
        got.append(int(tokens[down]))
        path.append(down)
        node = down
    total = torch.cumsum(r, 0)
    hit = (total > u[0] * total[-1]).nonzero()
    return got + [int(hit[0]) if len(hit) else -1], path
