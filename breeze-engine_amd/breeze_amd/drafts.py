"""Trees of drafted tokens on GPU tensors: several continuations of each sequence
in one pass of the target, between ``attention.kv_write`` and the next step.

- ``tree_attention``: attention of the trees' nodes over the cache;
- ``verify``: the drafted tokens against the target's logits with given random
  numbers, and the next token drawn, so that every token is distributed as the
  target's own (in place of the greedy token of ``hip_backend.matmul_argmax``);
- ``kv_compact``: the accepted nodes' cache rows moved together, in all layers.

A sequence's tree is its new tokens: node 0 is the last token that was decided,
whose key is not in the cache yet, the others are drafted.  ``parents``, int32
``[T]``, gives each node's parent by its number in its tree, a parent before its
children; -1, and anything that is not before the node, is no parent.  A tree has
at most 1024 nodes; a chain is a tree too, and so is a node alone.

The conventions are ``attention``'s: asynchronous calls on the current stream
that own no memory, shapes, types and strides checked here (``ValueError``), what
lies on the GPU bounded by the kernels, no gradients, no CPU fallback.
"""
import array

from . import attention as att
from . import hip_backend as hb


def tree_attention(q, cache, block_table, kv_lens, parents, cu_q=None, scale=None, out=None):
    """Attention of trees of drafted tokens over the cache; ``[T, heads, head_dim]``
    of q's type.

    As ``attention.paged_attention``, but for what a node sees: the keys before the
    tree, its ancestors and itself.  ``kv_lens`` counts the trees' nodes, whose keys
    are the sequence's last in the cache, node after node (``kv_write`` comes first).
    ``cu_q``: int32 ``[B + 1]``, where each sequence's nodes begin and the last one's
    end; None: one node a sequence.

    A row that sees no key is zero; rows of a tree past 1024 nodes are NaN; rows
    outside every sequence are not written.  Precision is ``paged_attention``'s, with
    two terms of fp16's weights at every length.  ``out`` may be given: q itself, or apart
    from it."""
    torch = att._torch()
    T, heads, D = q.shape if q.dim() == 3 else (0, 0, 0)
    if D != cache.head_dim or heads % cache.kv_heads or not heads:
        raise ValueError(f"q must be [T, a multiple of {cache.kv_heads} heads, {cache.head_dim}], got {tuple(q.shape)}")
    dt = att._type(q, "q")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, columns], got {tuple(block_table.shape)}")
    B, cols = block_table.shape
    att._ints(block_table, (B, cols), "block_table")
    att._ints(kv_lens, (B,), "kv_lens")
    att._ints(parents, (T,), "parents")
    if cu_q is not None:
        att._ints(cu_q, (B + 1,), "cu_q")
    elif T != B:
        raise ValueError(f"{T} nodes in {B} sequences: cu_q says where each begins")
    if scale is None:
        scale = D ** -0.5
    elif not 0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    att._same_device(cache._index, q, block_table, kv_lens, parents, cu_q, out)
    given = out is not None
    out = att._output(out, q, (T, heads, D), "out") if given else q.new_empty((T, heads, D))
    if T == 0 or B == 0:
        return out
    if cache._index != att._current():
        with torch.cuda.device(cache.device):
            return tree_attention(q, cache, block_table, kv_lens, parents, cu_q, scale, out)
    q = att._rows(q, "q")
    if given:
        att._no_overlap(out, q, "q")
    work, n = att._workspace((cache.kv_heads, cache.page_size, D, T, B, heads, dt, cols, cu_q is not None), "tree",
                             q.device)
    qs, os = q.stride(), out.stride()
    rc = hb._lib.i4_tree_attention_dev(
        cache._p, q.data_ptr(), qs[0], qs[1], T, heads, dt, block_table.data_ptr(), block_table.stride(0), cols,
        kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), B, parents.data_ptr(), scale, out.data_ptr(),
        os[0], os[1], None if work is None else work.data_ptr(), n, hb._torch_stream(q))
    if rc:
        hb._check_rc(rc, "i4_tree_attention_dev")
    return out


def _scores(t, T, V, what):
    if t.dim() != 2 or t.shape != (T, V):
        raise ValueError(f"{what} must be [{T}, {V}], got {tuple(t.shape)}")
    return t if t.stride(1) == 1 or V == 1 else t.contiguous()


def verify(logits, tokens, parents, uniforms, cu=None, temperature=1.0, draft=None, kv_lens=None):
    """Drafted tokens checked against the target, and the next one drawn;
    ``(new_tokens, path, counts)``.

    ``logits``: ``[T, V]``, at each node the scores of the token after it (fp32, bf16
    or fp16; -inf leaves a token out); ``tokens``: int32 ``[T]``, the nodes' own (node
    0's does not matter); ``uniforms``: fp32 ``[T]`` in [0, 1); ``cu``: int32 ``[B +
    1]``, where each sequence's nodes begin and the last one's end; None: one node a
    sequence, whose token is drawn.  ``temperature``: a number, or fp32 ``[B]``; 0 takes
    the largest score, the first of equal ones.  ``draft``: fp32 ``[T, V]``, at each
    node the probabilities (a row sums to 1) that its children were drawn with, one after
    another without the earlier ones; None: children that the draft did not draw (its
    best ones, say).  ``kv_lens``: int32 ``[B]``, as ``tree_attention`` had them: a negative
    one's sequence had no place in the cache (``PageTable.extend``), its scores mean
    nothing, and it gets no token, the count 0.

    From node 0 on, with r = softmax(logits / temperature) of the node, its children
    go in order: child c is taken where ``uniforms[c] * q(c) < r(c)``, q being 1
    without ``draft``, else ``draft`` over what it leaves without the earlier children;
    one that is not leaves r = max(r - q, 0) without it, normalized.  Where none is
    taken the next token is the first whose running sum of r passes ``uniforms`` of
    node 0.  So every token is distributed as the target's own.  All of it is worked
    out in 64 bits.

    ``counts``: int32 ``[B]``, the nodes on the path, node 0 among them, and as many new
    tokens: the accepted ones and then the drawn one.  ``path`` and ``new_tokens``: int32
    ``[T]``, packed like the nodes, -1 after the path's end.  A token that no
    distribution gives is -1 (a row with a NaN, +inf or nothing finite, a temperature
    below 0 or not finite, a draft that gives a child that it comes to NaN, infinity or
    less than 0, or NaN or infinity to any token after a rejected child); no node, or more
    than 1024, have the count 0.  A child whose token is not in the vocabulary, or an
    earlier sibling's, is passed over, and so is one that ``draft`` has nothing left for.
    Only rows of ``draft`` of nodes with children are read."""
    torch = att._torch()
    T, V = logits.shape if logits.dim() == 2 else (0, 0)
    if not 1 <= V <= 1 << 21:
        raise ValueError(f"logits must be [T, 1 to 2^21], got {tuple(logits.shape)}")
    dt = att._type(logits, "logits")
    logits = _scores(logits, T, V, "logits")
    if cu is None:
        B = T
    else:
        B = cu.shape[0] - 1 if cu.dim() == 1 else -1
        if B < 0:
            raise ValueError(f"cu must be [B + 1], got {tuple(cu.shape)}")
        att._ints(cu, (B + 1,), "cu")
    att._ints(tokens, (T,), "tokens")
    if parents is not None:
        att._ints(parents, (T,), "parents")
    elif cu is not None:
        raise ValueError("with cu, parents says how the nodes hang together")
    if kv_lens is not None:
        att._ints(kv_lens, (B,), "kv_lens")
    if uniforms.dtype is not torch.float32 or uniforms.shape != (T,) or (T > 1 and uniforms.stride(0) != 1):
        raise ValueError(f"uniforms must be contiguous float32 {(T,)}, got {uniforms.dtype} {tuple(uniforms.shape)}")
    temps = None
    if isinstance(temperature, torch.Tensor):
        temps, temperature = temperature, 0.0
        if temps.dtype is not torch.float32 or temps.shape != (B,) or (B > 1 and temps.stride(0) != 1):
            raise ValueError(f"temperature must be a number or contiguous float32 {(B,)}, got {temps.dtype} "
                             f"{tuple(temps.shape)}")
    elif not 0 <= temperature < 1e30:
        raise ValueError(f"temperature must be zero or more and finite, got {temperature}")
    if draft is not None:
        if draft.dtype is not torch.float32:
            raise ValueError(f"draft must be float32, got {draft.dtype}")
        draft = _scores(draft, T, V, "draft")
    index = logits.get_device()
    att._same_device(index, tokens, parents, uniforms, cu, temps, draft, kv_lens)
    if index != att._current():
        with torch.cuda.device(logits.device):
            return verify(logits, tokens, parents, uniforms, cu, temperature if temps is None else temps, draft, kv_lens)
    if B == 0:
        none = torch.full((2 * T,), -1, dtype=torch.int32, device=logits.device)
        return none[:T], none[T:], none[:0]
    new = tokens.new_empty((2 * T + B,))
    work, n = att._workspace((T, V, B, cu is not None, draft is not None), "verify", logits.device)
    p = new.data_ptr()
    rc = hb._lib.i4_verify_lens_dev(
        logits.data_ptr(), logits.stride(0), T, V, dt, tokens.data_ptr(), None if parents is None else parents.data_ptr(),
        uniforms.data_ptr(), None if cu is None else cu.data_ptr(), B, None if kv_lens is None else kv_lens.data_ptr(),
        None if temps is None else temps.data_ptr(), temperature, None if draft is None else draft.data_ptr(), 0 if draft is None else draft.stride(0), p, p + 4 * T,
        p + 8 * T, None if work is None else work.data_ptr(), n, hb._torch_stream(logits))
    if rc:
        hb._check_rc(rc, "i4_verify_lens_dev")
    return new.split((T, T, B))


def kv_compact(caches, block_table, kv_lens, cu_q, path, counts, lens=None):
    """The accepted nodes' cache rows moved together; the new lengths, int32 ``[B]``.

    ``caches``: a ``KVCache``, or a list of them (the layers'; of one geometry, with one
    ``block_table``), changed in place.  ``kv_lens``, ``cu_q``: as ``tree_attention``
    had them; ``path``, ``counts``: as ``verify`` gave them.  The row of node ``path[i]``
    goes to the place of node i, for the first ``counts`` of each sequence, and a
    sequence's length becomes the keys before its tree and those.  Rows past it keep what
    they hold.

    ``lens``: int32 ``[B]``, the lengths before the step (``PageTable.extend``'s): where
    kv_lens is negative nothing moves, and the sequence keeps that length, so that a
    later step can go on with it.  Without them its length becomes -1."""
    torch = att._torch()
    caches = [caches] if isinstance(caches, att.KVCache) else list(caches)
    if not 1 <= len(caches) <= 4096:
        raise ValueError(f"needs 1 to 4096 caches, got {len(caches)}")
    first = caches[0]
    for c in caches:
        if c._geometry != first._geometry:
            raise ValueError("the caches differ in pages, heads, sizes or device")
    if len({c._k for c in caches}) < len(caches):
        raise ValueError("a cache is given twice: its rows would move twice")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, columns], got {tuple(block_table.shape)}")
    B, cols = block_table.shape
    T = path.shape[0] if path.dim() else 0
    att._ints(block_table, (B, cols), "block_table")
    att._ints(kv_lens, (B,), "kv_lens")
    att._ints(path, (T,), "path")
    att._ints(counts, (B,), "counts")
    if cu_q is not None:
        att._ints(cu_q, (B + 1,), "cu_q")
    elif T != B:
        raise ValueError(f"{T} nodes in {B} sequences: cu_q says where each begins")
    if lens is not None:
        att._ints(lens, (B,), "lens")
    att._same_device(first._index, block_table, kv_lens, cu_q, path, counts, lens)
    if first._index != att._current():
        with torch.cuda.device(first.device):
            return kv_compact(caches, block_table, kv_lens, cu_q, path, counts, lens)
    after = kv_lens.new_empty((B,))
    if B:
        pointers = array.array("Q", [c._p for c in caches])  # the C structs' addresses; a ctypes array takes longer to fill
        rc = hb._lib.i4_kv_compact_lens_dev(
            pointers.buffer_info()[0], len(caches), block_table.data_ptr(), block_table.stride(0), cols, kv_lens.data_ptr(),
            None if lens is None else lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), T, B, path.data_ptr(),
            counts.data_ptr(), after.data_ptr(), hb._torch_stream(after))
        if rc:
            hb._check_rc(rc, "i4_kv_compact_lens_dev")
    return after
