"""A decode step with drafted tokens over the quantized paged cache, as timed cases.

Each case is one call (or one pair of calls) of ``breeze_amd.attention`` or
``breeze_amd.drafts`` on GPU tensors:

- ``rope``: rotary positions of queries and keys that are columns of one fused
  projection;
- ``pages``: new tokens' pages, slots, positions and lengths worked out on the
  GPU from the requests' lengths, and the pages given back;
- ``tree``: attention of a tree of drafted tokens a sequence over the cache, in
  which a token sees the cached ones before the tree, its ancestors and itself;
- ``verify``: the drafted tokens checked against the target's logits with given
  random numbers, down the tree, and the next token drawn;
- ``compact``: the accepted tokens' cache rows moved to consecutive places, in
  all layers.

A tree's nodes are packed row by row like the tokens of other calls; ``parents``
gives each node's parent by its number in its tree (-1: none), parents first.
Node 0 is the last token that was decided, the others are drafted.

``lens`` and ``ctx`` give the new and the cached tokens of each sequence:
``"5,1,77"`` one by one, ``"64x1"`` that many alike, ``"64x1-8000"`` that many
spread over the logarithm (with ``spread``, the seed of that spread).
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_KV = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


_modules = None


def _framework():
    """The modules ``attention`` and ``drafts``."""
    global _modules
    if _modules is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "breeze-engine_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from breeze_amd import attention, drafts

        _modules = attention, drafts
    return _modules


# ------------------------------------------------------------------ cases

def _rope(tokens, heads, kv_heads, dim, rotary, layout, scaling, start, dtype):
    return dict(op="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, layout=layout,
                scaling=scaling, start=start, dtype=dtype)


def _pages(lens, ctx, page, chain, spread=0):
    return dict(op="pages", lens=lens, ctx=ctx, page=page, chain=chain, spread=spread)


def _tree(lens, ctx, heads, kv_heads, dim, page, kind, dtype, spread=0):
    return dict(op="tree", lens=lens, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind,
                dtype=dtype, spread=spread)


def _verify(lens, vocab, draft, temperature, dtype, spread=0):
    return dict(op="verify", lens=lens, vocab=vocab, draft=draft, temperature=temperature, dtype=dtype, spread=spread)


def _compact(lens, ctx, layers, kv_heads, dim, page, kind, spread=0):
    return dict(op="compact", lens=lens, ctx=ctx, layers=layers, kv_heads=kv_heads, dim=dim, page=page, kind=kind,
                spread=spread)


def listed():
    return [
        # One decode step's token, the full-attention layers' heads of the 27B decoder, a quarter of
        # each turned: latency.
        dict(_rope(1, 24, 4, 256, 64, "half", "none", 4100, "fp32"), name="rope_one"),
        # A long prompt's last chunk, whole heads, far positions.
        dict(_rope(8192, 32, 8, 128, 128, "interleaved", "parts", 122880, "bf16"), name="rope_prompt"),
        # A serving batch's step: a tree of drafted tokens for each of 64 requests of very different lengths.
        dict(_pages("64x16", "64x100-16000", 16, False, spread=3), name="pages_batch"),
        # Prompts of odd lengths that come in together.
        dict(_pages("5000,1,777,4097,33,2500,1234", "0,40,0,3,1000,0,517", 16, True), name="pages_prompts"),
        # One sequence with a small tree: latency.
        dict(_tree("12", "4100", 24, 4, 256, 16, "int8", "fp32"), name="tree_one"),
        # A serving batch of trees over contexts of very different lengths.
        dict(_tree("16x32", "16x500-8000", 32, 8, 128, 16, "fp8", "bf16", spread=3), name="tree_batch"),
        # A large tree behind a long context.
        dict(_tree("61", "31744", 32, 8, 128, 64, "int8", "fp16"), name="tree_long"),
        # One sequence's small tree against the 27B decoder's vocabulary, drafted tokens without
        # probabilities of their own.
        dict(_verify("12", 151936, False, 0.8, "fp32"), name="verify_one"),
        # A serving batch of trees.
        dict(_verify("40x16", 151936, False, 0.7, "fp32"), name="verify_batch"),
        # Chains of odd lengths drawn from a draft's probabilities, an odd vocabulary.
        dict(_verify("24x3-9", 32003, True, 1.0, "bf16", spread=5), name="verify_drawn"),
        # One sequence's accepted tokens in the sixteen full-attention layers of the 27B decoder.
        dict(_compact("25", "4100", 16, 4, 256, 16, "int8"), name="compact_one"),
        # A serving batch, several layers.
        dict(_compact("48x32", "48x100-4000", 8, 8, 128, 16, "fp8", spread=3), name="compact_batch"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


_HEADS = [(24, 4, 256), (32, 8, 128), (16, 2, 64), (8, 8, 128)]


def draw(rng):
    op = rng.choice(["rope", "pages", "tree", "tree", "tree", "verify", "verify", "compact"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    page, kind, spread = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "fp8"]), rng.randrange(1 << 20)
    heads, kv_heads, dim = rng.choice(_HEADS)
    if op == "rope":
        rotary = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randrange(1, dim // 2 + 1)])
        tokens = _log(rng, 1, 8192 if dim < 256 else 4096)
        return _rope(tokens, heads, kv_heads, dim, rotary, rng.choice(["half", "interleaved"]),
                     rng.choice(["none", "linear", "base", "parts"]), _log(rng, 1, 200000), dtype)
    if op == "pages":
        n = _log(rng, 1, 256)
        hi = _log(rng, 2, 16384 // n)
        chain = hi > 64 or rng.random() < 0.5
        return _pages("%dx1-%d" % (n, hi), "%dx1-%d" % (n, _log(rng, 1, 16000)), page, chain, spread)
    if op == "tree":
        n = _log(rng, 1, 32)
        hi = _log(rng, 1, min(100, 512 // n))
        ctx = _log(rng, 1, min(32000, 128000 // n, 1300000 // (n * hi)))
        return _tree("%dx1-%d" % (n, hi), "%dx1-%d" % (n, ctx), heads, kv_heads, dim, page, kind, dtype, spread)
    if op == "verify":
        vocab = rng.choice([151936, _log(rng, 1000, 151936)])
        n, draft = _log(rng, 1, 64), rng.random() < 0.4
        hi = _log(rng, 1, min(60, (300 if draft else 600) // n))
        return _verify("%dx1-%d" % (n, hi), vocab, draft, rng.choice([0.0, 0.6, 0.8, 1.0]), dtype, spread)
    n = _log(rng, 1, 48)
    return _compact("%dx2-%d" % (n, _log(rng, 2, 64)), "%dx1-%d" % (n, _log(rng, 1, 4000)), rng.choice([1, 4, 8]),
                    kv_heads, dim, page, kind, spread)


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
    n = _lens(case["lens"], rng)
    return n, (_lens(case["ctx"], rng) if "ctx" in case else [0] * len(n))


# ------------------------------------------------------------------ inputs

class _State:
    pass


def _parents(lens, rng, chain=False):
    """Trees in the order of their levels, up to four children a node."""
    out = []
    for n in lens:
        for i in range(n):
            if chain or i < 2:
                out.append(i - 1)
            else:
                out.append(max(out[-1], rng.randrange(max(0, (i - 1) // 4), (i + 1) // 2)))
    return out


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _quantized(x, kind):
    """Cache bytes and scales of fp32 rows [..., D]."""
    top = x.abs().amax(-1).clamp_min(1e-20)
    if kind == "int8":
        scale = top / 127
        return (x / scale.unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8), scale
    scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
    return (x / scale.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8), scale


def _paged(s, case, gen):
    """A block table over pages in any order; the number of pages."""
    page = case["page"]
    s.lens, s.ctx = _shape(case)
    s.cu = _cu(s.lens)
    s.kv_lens = torch.tensor([c + n for c, n in zip(s.ctx, s.lens)], dtype=torch.int32, device="cuda")
    need = [(c + n + page - 1) // page for c, n in zip(s.ctx, s.lens)]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    s.table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        s.table[b, :n] = order[at:at + n]
        at += n
    return pages


def _filled(case, pages, gen):
    """Cache tensors k, v, k_scale, v_scale: channels of unlike size, as projections give them."""
    H, page, D, kind = case["kv_heads"], case["page"], case["dim"], case["kind"]
    out = [torch.empty((pages, H, page, D), dtype=torch.int8, device="cuda") for _ in range(2)]
    out += [torch.empty((pages, H, page), dtype=torch.float32, device="cuda") for _ in range(2)]
    for i in range(2):
        bias = torch.exp(0.5 * torch.randn((H, 1, D), generator=gen, device="cuda"))
        for p in range(0, pages, 4096):
            part = torch.randn((min(4096, pages - p), H, page, D), generator=gen, device="cuda") * bias
            out[i][p:p + 4096], out[2 + i][p:p + 4096] = _quantized(part, kind)
    return [x.view(_KV[kind]) for x in out[:2]] + out[2:]


_BASE, _FACTOR, _ORIGINAL = 1e6, 8.0, 16384


def _frequencies(rotary, scaling):
    """Radians a position, in 64 bits, and the amplitude."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda")
    base = _BASE
    if scaling == "base" and rotary > 2:
        base = _BASE * _FACTOR ** (rotary / (rotary - 2))
    f = base ** (-i / rotary)
    if scaling == "linear":
        return f / _FACTOR, 1.0
    if scaling == "parts":  # as they are where they turn often in the original context, divided where hardly ever
        keep = ((_ORIGINAL * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        return f * (keep + (1 - keep) / _FACTOR), 0.1 * math.log(_FACTOR) + 1
    return f, 1.0


def _prepare_rope(s, case, gen):
    T, Hq, Hk, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    # One projection's columns: queries, keys and the values behind them.
    qkv = torch.randn((T, (Hq + 2 * Hk) * D), generator=gen, device="cuda").to(_DT[case["dtype"]])
    s.q, s.k, _ = (x.view(T, -1, D) for x in qkv.split([Hq * D, Hk * D, Hk * D], dim=1))
    s.positions = (torch.arange(T, device="cuda") + case["start"]).to(torch.int32)
    s.freqs, s.amplitude = _frequencies(case["rotary"], case["scaling"])


def _prepare_pages(s, case, gen):
    page = case["page"]
    s.lens, s.ctx = _shape(case)
    B = len(s.lens)
    s.cu, s.ctx_lens = _cu(s.lens), torch.tensor(s.ctx, dtype=torch.int32, device="cuda")
    parents = _parents(s.lens, random.Random(case["spread"]), case["chain"])
    s.parents = None if case["chain"] else torch.tensor(parents, dtype=torch.int32, device="cuda")
    held = [(c + page - 1) // page for c in s.ctx]
    need = [(c + n + page - 1) // page for c, n in zip(s.ctx, s.lens)]
    # Half of the batches come to a cache that has no room for all of them.
    total = sum(need) + 5
    if random.Random(B + sum(s.lens)).random() < 0.5:
        total = sum(held) + (sum(need) - sum(held)) * 3 // 4 + 1
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    s.table = torch.full((B, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        s.table[b, :n] = order[at:at + n]
        at += n
    s.held = torch.tensor(held, dtype=torch.int32, device="cuda")
    s.free = torch.zeros((total,), dtype=torch.int32, device="cuda")
    s.free[:total - at] = order[at:]
    s.count = torch.tensor([total - at], dtype=torch.int32, device="cuda")


def _prepare_tree(s, case, gen):
    pages = _paged(s, case, gen)
    s.cache = _filled(case, pages, gen)
    s.parents = torch.tensor(_parents(s.lens, random.Random(case["spread"])), dtype=torch.int32, device="cuda")
    T = sum(s.lens)
    s.q = (1.5 * torch.randn((T, case["heads"], case["dim"]), generator=gen, device="cuda")).to(_DT[case["dtype"]])


def _prepare_verify(s, case, gen):
    s.lens, _ = _shape(case)
    T, V = sum(s.lens), case["vocab"]
    parents = _parents(s.lens, random.Random(case["spread"]), case["draft"])
    s.parents, s.cu = torch.tensor(parents, dtype=torch.int32, device="cuda"), _cu(s.lens)
    # A language model's scores: a few tokens stand out of many.
    x = 3 * torch.randn((T, V), generator=gen, device="cuda")
    at = torch.randint(V, (T, 4), generator=gen, device="cuda")
    x.scatter_add_(1, at, 6 + 8 * torch.rand((T, 4), generator=gen, device="cuda"))
    s.logits = x.to(_DT[case["dtype"]])
    # The draft sees nearly the same scores.
    x += 0.7 * torch.randn((T, V), generator=gen, device="cuda")
    s.draft = None
    if case["draft"]:
        s.draft = torch.softmax(x, dim=-1)
        x -= torch.log(-torch.log(torch.rand((T, V), generator=gen, device="cuda").clamp_(1e-9, 1 - 1e-7)))
    best = x.topk(4, dim=-1).indices.tolist()
    # A node's token is its parent's next best, or next drawn, one.
    tokens, start = [], 0
    for n in s.lens:
        children = {}
        for i in range(n):
            p = parents[start + i]
            k = children[p] = children.get(p, -1) + 1
            tokens.append(best[start + p][k % 4] if p >= 0 else 0)
        start += n
    s.tokens = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    s.uniforms = torch.rand((T,), generator=gen, device="cuda")
    s.temperature = torch.full((len(s.lens),), case["temperature"], dtype=torch.float32, device="cuda")


def _depths(parents, lens):
    out, start = [], 0
    for n in lens:
        for i in range(n):
            p = parents[start + i]
            out.append(out[start + p] + 1 if p >= 0 else 0)
        start += n
    return out


def _prepare_compact(s, case, gen):
    pages = _paged(s, case, gen)
    H, page, D = case["kv_heads"], case["page"], case["dim"]
    # All layers' pages in one allocation of each kind, as a program makes them.
    shape = (case["layers"], pages, H, page)
    s.pages = [torch.randint(-120, 120, (*shape, D), dtype=torch.int8, generator=gen, device="cuda") for _ in range(2)]
    s.pages += [torch.rand(shape, generator=gen, device="cuda") for _ in range(2)]
    s.layers = [[x[i].view(_KV[case["kind"]]) if x.dim() == 5 else x[i] for x in s.pages] for i in range(case["layers"])]
    # A path down each tree: its nodes' numbers grow, and lie past the places that they move to, so that
    # the same call again leaves what the first did.
    rng = random.Random(case["spread"] + int(torch.randint(1 << 30, (1,), generator=gen, device="cuda")))
    path, counts = [], []
    for n in s.lens:
        m = rng.randrange(0, min(6, n // 2 - 1) + 1) if n > 3 else rng.randrange(n)
        nodes = [0] + (sorted(rng.sample(range(m + 1, n), m)) if n > 3 else list(range(1, m + 1)))
        path += nodes + [-1] * (n - len(nodes))
        counts.append(len(nodes))
    s.path = torch.tensor(path, dtype=torch.int32, device="cuda")
    s.counts = torch.tensor(counts, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 29)
    s = _State()
    s.case = case
    s.handle = None  # the object that a program makes once: a cache, a page table, a rotary's frequencies
    {"rope": _prepare_rope, "pages": _prepare_pages, "tree": _prepare_tree, "verify": _prepare_verify,
     "compact": _prepare_compact}[case["op"]](s, case, gen)
    return s


# ------------------------------------------------------------------ one pass

def _run_own(s):
    att, drafts = _framework()
    c = s.case
    if c["op"] == "rope":
        if s.handle is None:
            more = {} if c["scaling"] == "none" else dict(scaling=c["scaling"], factor=_FACTOR)
            if c["scaling"] == "parts":
                more["original"] = _ORIGINAL
            s.handle = att.Rotary(c["rotary"], base=_BASE, layout=c["layout"], **more)
        return att.rotary(s.handle, s.q, s.k, s.positions)
    if c["op"] == "pages":
        if s.handle is None:
            s.handle = att.PageTable(s.table, s.held, s.free, s.count, c["page"])
        got = s.handle.extend(s.ctx_lens, s.cu, sum(s.lens), s.parents)
        s.handle.trim(s.ctx_lens)
        return (*got, s.table, s.held, s.free, s.count)
    if c["op"] == "tree":
        if s.handle is None:
            s.handle = att.KVCache(*s.cache)
        return drafts.tree_attention(s.q, s.handle, s.table, s.kv_lens, s.parents, s.cu)
    if c["op"] == "verify":
        return drafts.verify(s.logits, s.tokens, s.parents, s.uniforms, s.cu, s.temperature, s.draft)
    if s.handle is None:
        s.handle = [att.KVCache(*layer) for layer in s.layers]
    lens = drafts.kv_compact(s.handle, s.table, s.kv_lens, s.cu, s.path, s.counts)
    return lens, s.pages


def _run_rope(s):
    c = s.case
    angle = s.positions.double()[:, None] * s.freqs
    cos, sin = ((f(angle) * s.amplitude).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    out = []
    for x in (s.q, s.k):
        y = x.float().clone()
        part = y[..., :c["rotary"]]
        a, b = (part[..., 0::2], part[..., 1::2]) if c["layout"] == "interleaved" else part.chunk(2, dim=-1)
        turned = a * cos - b * sin, b * cos + a * sin
        a.copy_(turned[0])
        b.copy_(turned[1])
        out.append(y.to(x.dtype))
    return tuple(out)


def _ancestors(s):
    """[T, n]: whether node j of its tree is an ancestor of a node, or itself; and the nodes' depths."""
    n = max(s.lens)
    start = torch.repeat_interleave(s.cu[:-1], s.cu[1:] - s.cu[:-1], output_size=sum(s.lens)).long()
    me = torch.arange(start.shape[0], device="cuda") - start
    up = torch.zeros((start.shape[0], n + 1), dtype=torch.bool, device="cuda")
    at, depth = me, torch.full_like(me, -1)
    for _ in range(s.deepest):
        up.scatter_(1, torch.where(at >= 0, at, n).unsqueeze(1), True)
        depth += at >= 0
        at = torch.where(at >= 0, s.parents.long()[start + at.clamp_min(0)], -1)
    return up[:, :n], depth


def _deepest(s):
    if not hasattr(s, "deepest"):
        s.deepest = 1 + max(_depths(s.parents.tolist(), s.lens))


def _run_pages(s):
    page, B, cols = s.case["page"], s.table.shape[0], s.table.shape[1]
    n = s.cu[1:] - s.cu[:-1]
    end = s.ctx_lens + n
    want = (end + page - 1) // page
    fits = want <= cols
    need = torch.where(fits, (want - s.held).clamp_min(0), 0)
    until = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (until <= s.count))
    need = torch.where(ok, need, 0)
    col = torch.arange(cols, device="cuda") - s.held[:, None]  # which of a sequence's new pages a column takes
    new = (col >= 0) & (col < need[:, None])
    at = s.count - 1 - ((until - need)[:, None] + col)
    s.table.copy_(torch.where(new, s.free[at.clamp(0, s.free.shape[0] - 1).long()], s.table))
    s.held += need
    s.count -= need.sum()
    kv_lens = torch.where(ok, end, -1).to(torch.int32)
    # The new tokens' places.
    T = sum(s.lens)
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), n, output_size=T)
    i = torch.arange(T, device="cuda") - s.cu[seq]
    place = s.ctx_lens[seq] + i
    slots = s.table[seq, (place // page).clamp_max(cols - 1).long()] * page + place % page
    slots = torch.where(ok[seq], slots, -1).to(torch.int32)
    if s.parents is not None:
        _deepest(s)
        place = s.ctx_lens[seq] + _ancestors(s)[1]
    positions = place.to(torch.int32)
    # And back.
    keep = torch.minimum((s.ctx_lens + page - 1) // page, s.held)
    gone = s.held - keep
    first = torch.cumsum(gone, 0) - gone
    col = torch.arange(cols, device="cuda") - keep[:, None]
    old = (col >= 0) & (col < gone[:, None])
    total = gone.sum()
    at = s.count + total - 1 - (first[:, None] + col)
    room = torch.cat([s.free, s.free[:1]])
    room[torch.where(old, at, s.free.shape[0]).long()] = s.table
    s.free.copy_(room[:-1])
    s.table.masked_fill_(old, -1)
    s.held.copy_(keep)
    s.count += total
    return slots, positions, kv_lens, s.table, s.held, s.free, s.count


def _padded(cu, n):
    """Row numbers of the packed nodes, [sequences, n], and which are real."""
    at = cu[:-1, None].long() + torch.arange(n, device=cu.device)
    real = at < cu[1:, None]
    return torch.where(real, at, 0), real


def _run_tree(s):
    c = s.case
    page, Hq, H, D = c["page"], c["heads"], c["kv_heads"], c["dim"]
    B, G, n = len(s.lens), c["heads"] // c["kv_heads"], max(s.lens)
    keys = max(a + b for a, b in zip(s.lens, s.ctx))
    at, real = _padded(s.cu, n)
    q = s.q.float()[at].view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    j = torch.arange(keys, device="cuda")
    where = (s.table.long()[:, j // page].clamp_min(0), slice(None), j % page)

    def gathered(i):  # [B, H, keys, D]
        x = s.cache[i].view(torch.int8)[where].view(_KV[c["kind"]]).float() * s.cache[2 + i][where].unsqueeze(-1)
        return x.permute(0, 2, 1, 3)

    scores = torch.matmul(q, gathered(0).transpose(2, 3).contiguous()).view(B, H, G, n, keys) / math.sqrt(D)
    # A node sees the tokens before the tree, and in the tree its ancestors and itself.
    _deepest(s)
    up = _ancestors(s)[0][at]  # [B, n, n]
    node = (j - (s.kv_lens - (s.cu[1:] - s.cu[:-1]))[:, None])[:, None].expand(B, n, keys)
    seen = (node < 0) | ((node < n) & torch.gather(up, 2, node.clamp(0, n - 1)))
    seen &= real[:, :, None] & (j < s.kv_lens[:, None])[:, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, H, G * n, keys), gathered(1).contiguous()).view(B, H, G, n, D)
    out = out / total.clamp_min(1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[real].to(s.q.dtype)


def _run_verify(s):
    """All sequences go down their trees together, in 64 bits: a random number may fall next to a border."""
    T, V = s.logits.shape
    B = len(s.lens)
    if not hasattr(s, "most"):
        parents = s.parents.tolist()
        s.deepest = 1 + max(_depths(parents, s.lens))
        ends, s.most, start = [], 0, 0
        for n in s.lens:
            mine = parents[start:start + n]
            s.most = max([s.most] + [mine.count(p) for p in range(n)])
            start += n
    first, end = s.cu[:-1].long(), s.cu[1:].long()
    row = torch.arange(T, device="cuda")
    start = torch.repeat_interleave(first, end - first, output_size=T)
    parent = torch.where(s.parents >= 0, start + s.parents, -1)
    tokens = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    path = torch.full((T + 1,), -1, dtype=torch.int32, device="cuda")  # the last place takes what is not written
    path[first] = 0
    counts = torch.ones((B,), dtype=torch.int64, device="cuda")
    cur, going = first.clone(), torch.ones((B,), dtype=torch.bool, device="cuda")
    last = torch.zeros((B, V), dtype=torch.float64, device="cuda")
    u_all, t = s.uniforms.double(), s.temperature.double()[:, None]
    greedy = t == 0
    seqs = torch.arange(B, device="cuda")
    for _ in range(s.deepest):
        l = s.logits[cur].double()
        top, best = l.max(-1, keepdim=True)
        p = torch.exp((l - top) / torch.where(greedy, 1.0, t))
        p = torch.where(greedy, (torch.arange(V, device="cuda") == best).double(), p / p.sum(-1, keepdim=True))
        q = None if s.draft is None else s.draft[cur].double()
        G, S = p.clone(), torch.ones((B,), dtype=torch.float64, device="cuda")
        A, Q = torch.zeros_like(S), torch.ones_like(S)
        found = torch.full((B,), -1, dtype=torch.int64, device="cuda")
        is_child = parent[None] == cur[:, None]  # [B, T]
        rank = torch.cumsum(is_child, 1)
        for k in range(s.most):
            hit = is_child & (rank == k + 1)
            has = hit.any(1) & (found < 0)
            child = hit.to(torch.int8).argmax(1)
            token = s.tokens[child].long()
            prob = 1.0 if q is None else q[seqs, token] / Q
            accept = has & (u_all[child] * prob * S < G[seqs, token])
            found = torch.where(accept, child, found)
            reject = has & ~accept
            p[seqs, token] = torch.where(reject, 0.0, p[seqs, token])
            if q is None:
                G = p
            else:
                A = torch.where(reject, A + S / Q, A)
                G = (p - A[:, None] * q).clamp_min(0)
                Q = torch.where(reject, Q - q[seqs, token], Q)
            S = torch.where(reject, G.sum(-1), S)
        stop = going & (found < 0)
        last = torch.where(stop[:, None], G, last)
        going = going & (found >= 0)
        at = torch.where(going, first + counts, T)
        path[at] = torch.where(going, found - first, -1).to(torch.int32)
        counts += going
        cur = torch.where(going, found, cur)
    # Accepted tokens, then the drawn one: the first whose running sum passes the random number.
    until = torch.cumsum(last, -1)
    drawn = (until <= (u_all[first] * until[:, -1])[:, None]).sum(-1)
    path = path[:T]
    i = row - start
    n = counts[torch.repeat_interleave(seqs, end - first, output_size=T)]
    node = path[(row + 1).clamp_max(T - 1)].long()
    tokens = torch.where(i + 1 < n, s.tokens[(start + node).clamp(0, T - 1)], -1)
    tokens[first + counts - 1] = drawn.to(torch.int32)
    return tokens, path, counts.to(torch.int32)


def _run_compact(s):
    page, T = s.case["page"], s.path.shape[0]
    n = (s.cu[1:] - s.cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.shape[0], device="cuda"), n, output_size=T)
    i = torch.arange(T, device="cuda") - s.cu[seq]
    ctx = (s.kv_lens - n)[seq]
    keep = i < s.counts[seq]
    slot = []
    for place in (ctx + torch.where(keep, s.path, i), ctx + i):  # what is not kept moves to where it is
        slot.append((s.table[seq, (place // page).long()].long(), place % page))
    (p0, r0), (p1, r1) = slot
    for layer in s.layers:
        for x in layer:
            x = x.view(torch.int8) if x.dim() == 4 else x
            moved = torch.where(keep.view(-1, *[1] * (x.dim() - 2)), x[p0, :, r0], x[p1, :, r1])
            x[p1, :, r1] = moved
    lens = (s.kv_lens - n + s.counts).to(torch.int32)
    return lens, s.pages


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _run_rope, "pages": _run_pages, "tree": _run_tree, "verify": _run_verify,
            "compact": _run_compact}[s.case["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * e + 4 * case["tokens"], "flops": 3 * n * case["rotary"]}
    lens, ctx = _shape(case)
    T, B = sum(lens), len(lens)
    if case["op"] == "pages":
        page = case["page"]
        new = sum((c + n + page - 1) // page - (c + page - 1) // page for n, c in zip(lens, ctx))
        # Slots and positions out; new pages off the stack and back, into the table and out of it.
        return {"bytes": 8 * T + (0 if case["chain"] else 4 * T) + 16 * new + 24 * B, "flops": T}
    if case["op"] == "verify":
        return {"bytes": T * case["vocab"] * (e + (4 if case["draft"] else 0)) + 24 * T, "flops": 4 * T * case["vocab"]}
    D, H = case["dim"], case["kv_heads"]
    if case["op"] == "compact":
        rows = case["layers"] * 2 * H * B * 3  # three tokens a sequence, say
        return {"bytes": 2 * rows * (D + 4) + 4 * T + 20 * B, "flops": rows}
    kv = T + sum(ctx)
    pairs = sum(n * c + n * (n + 3) // 4 for n, c in zip(lens, ctx))
    b = 2 * T * case["heads"] * D * e + 2 * kv * H * (D + 4) + 4 * kv // case["page"] + 4 * T
    return {"bytes": b, "flops": 4 * D * case["heads"] * pairs}


# ------------------------------------------------------------------ in 64 bits

def _exact_rope(s, c):
    """Each pair as a complex number times e^(i angle)."""
    turn = s.amplitude * torch.exp(1j * s.positions.double()[:, None, None] * s.freqs)
    half, r = c["rotary"] // 2, c["rotary"]
    out = []
    for x in (s.q, s.k):
        y = x.double().clone()
        if c["layout"] == "half":
            z = torch.complex(y[..., :half].contiguous(), y[..., half:r].contiguous()) * turn
            y[..., :half], y[..., half:r] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :r].reshape(*y.shape[:2], half, 2).contiguous()) * turn
            y[..., :r] = torch.view_as_real(z).reshape(*y.shape[:2], r)
        out.append(y)
    return tuple(out)


def _exact_tree(s, c):
    H, G, page, D = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"], c["dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    parents = s.parents.tolist()
    start = 0
    for b, (n, ctx) in enumerate(zip(s.lens, s.ctx)):
        keys = ctx + n
        pages = s.table[b, :(keys + page - 1) // page].long()
        hidden = torch.zeros((n, keys), dtype=torch.bool)
        hidden[:, ctx:] = True
        for i in range(n):
            j = i
            while j >= 0:
                hidden[i, ctx + j] = False
                j = parents[start + j]
        hidden = hidden.to("cuda")
        for h in range(H):
            k, v = (s.cache[i].view(torch.int8)[pages, h].view(_KV[c["kind"]]).double().reshape(-1, D)[:keys]
                    * s.cache[2 + i][pages, h].double().reshape(-1, 1)[:keys] for i in range(2))
            for g in range(h * G, h * G + G):
                x = s.q[start:start + n, g].double() @ k.t() * D ** -0.5
                out[start:start + n, g] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v
        start += n
    return out


def _exact_verify(s, c):
    """One sequence after another, each rejected sibling's residual normalized in turn."""
    parents, given, u = s.parents.tolist(), s.tokens.tolist(), s.uniforms.double().tolist()
    tokens, path, counts = [], [], []
    start = 0
    for n in s.lens:
        node, nodes, got = 0, [0], []
        while True:
            l = s.logits[start + node].double()
            if c["temperature"] == 0:
                r = torch.zeros_like(l)
                r[int(torch.argmax(l))] = 1.0
            else:
                r = torch.softmax(l / s.temperature[0].double(), dim=-1)
            q = None if s.draft is None else s.draft[start + node].double().clone()
            left, down = 1.0, -1
            for i in range(node + 1, n):
                if parents[start + i] != node:
                    continue
                x = given[start + i]
                if u[start + i] * (1.0 if q is None else float(q[x]) / left) < float(r[x]):
                    down = i
                    break
                if q is not None:
                    rest = (r - q / left).clamp_min(0)
                    left -= float(q[x])
                    q[x] = 0.0
                else:
                    rest = r.clone()
                rest[x] = 0.0
                r = rest / rest.sum()
            if down < 0:
                break
            nodes.append(down)
            got.append(given[start + down])
            node = down
        total = torch.cumsum(r, 0)
        got.append(int(torch.searchsorted(total, (u[start] * total[-1]).reshape(1), right=True)))
        tokens += got + [-1] * (n - len(got))
        path += nodes + [-1] * (n - len(nodes))
        counts.append(len(nodes))
        start += n
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (tokens, path, counts))


def exact(case, seed):
    if case["op"] in ("pages", "compact"):  # whole numbers and moved rows
        return None
    s = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "verify": _exact_verify}[case["op"]](s, case)
