"""The decoder's token mixers on GPU tensors: what runs between a layer's
quantized projections (``hip_backend``).

- ``KVCache`` holds one layer's keys and values in pages, as INT8 or e4m3 with
  one scale for each token and head; ``kv_write`` quantizes new tokens into it
  and ``kv_read`` reads tokens back.
- ``paged_attention``: causal attention of new tokens (one a sequence, or a
  chunk) over that cache, in place of the decoder's full attention
  (kernel/qwen35_decoder.cpp:334-395, which keeps fp32 keys and values).
- ``gated_linear_attention``: the linear-attention layers' recurrence
  (kernel/qwen35_decoder.cpp:46-121), one token at a time from a kept state or
  whole prompts in chunks.

Tensors are fp32, bf16 or fp16 on one gfx950 GPU.  Calls are asynchronous on
the current stream, own no memory between calls (a workspace comes from
torch's allocator) and can be captured into graphs.  Shapes, types and strides
are checked here and raise ``ValueError``; what lies on the GPU (lengths,
offsets, page and slot numbers) is checked by the kernels, which skip what is
out of range.  Outputs carry no gradient.  There is no CPU fallback.
"""
import ctypes

from . import hip_backend as hb

_dtypes = None  # torch dtype -> the library's number for it
_current = None  # the current device's index


class _CCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("num_pages", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("page_size", ctypes.c_int), ("head_dim", ctypes.c_int), ("kind", ctypes.c_int)]


def _torch():
    global _dtypes, _current
    torch = hb._torch
    if torch is None or _dtypes is None:
        torch = hb._import_torch()
        _current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        _dtypes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    return torch


def _type(t, what):
    n = _dtypes.get(t.dtype)
    if n is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return n


def _rows(t, what):
    """`t` [T, heads, D] with its last dimension contiguous and rows that the
    kernels' wide loads can read: itself, or a copy."""
    st = t.stride()
    if st[2] == 1 and not (st[0] | st[1]) & 3 and not t.data_ptr() & 15:
        return t
    # A new tensor in any case: contiguous() gives one token back as it is, whose stride does not count.
    return t.clone(memory_format=_torch().contiguous_format)


def _ints(t, shape, what):
    if t.dtype is not hb._torch.int32 or t.shape != shape or (shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what} must be int32 of shape {shape} with a contiguous last dimension, "
                         f"got {t.dtype} {tuple(t.shape)} (strides {t.stride()})")
    return t


def _same_device(index, *tensors):
    """All tensors lie on GPU `index` (-1: a tensor that is not on one)."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"a tensor lies on {t.device}: all must be on one GPU")
    if index < 0:
        raise ValueError("tensors must be on a GPU")
    if hb._lib is None:
        hb._require_lib()


def _workspace(shape, kind, device):
    """(tensor or None, bytes) of a call's workspace; what a shape needs is asked once."""
    key = (kind, device.index, shape)
    n = _needs.get(key)
    if n is None:
        query = (hb._lib.i4_paged_attention_workspace if kind == "paged"
                 else hb._lib.i4_gated_linear_attention_workspace)
        n = query(*shape)
        if n < 0:
            raise ValueError(hb.last_error())
        if len(_needs) >= 4096:
            _needs.clear()
        _needs[key] = n
    return (hb._torch.empty((n,), dtype=hb._torch.uint8, device=device) if n else None), n


_needs = {}


class KVCache:
    """One layer's keys and values in pages.

    ``k``, ``v``: ``[pages, kv_heads, page_size, head_dim]``, int8 or
    float8_e4m3fn; ``k_scale``, ``v_scale``: fp32 ``[pages, kv_heads,
    page_size]``.  A value is the stored number times its token's and head's
    scale.  ``head_dim`` is 64, 128 or 256; ``page_size`` a power of two from 16
    to 1024.  The tensors are kept as given and written in place.  A token's row
    that attention may see has been written by ``kv_write``; what unwritten rows
    hold does not matter."""

    def __init__(self, k, v, k_scale, v_scale):
        torch = _torch()
        kinds = {torch.int8: 0, torch.float8_e4m3fn: 1}
        if k.dtype not in kinds or v.dtype is not k.dtype:
            raise ValueError(f"cache pages must be int8 or float8_e4m3fn, both alike, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"cache pages must be [pages, kv_heads, page_size, head_dim], both alike, got "
                             f"{tuple(k.shape)} and {tuple(v.shape)}")
        P, H, page, D = k.shape
        if D not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {D}")
        if page & (page - 1) or not 16 <= page <= 1024:
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page}")
        if P < 1 or not 1 <= H <= 4096 or P * page >= 1 << 31:
            raise ValueError(f"a cache needs a page, 1 to 4096 heads and fewer than 2^31 slots, got {tuple(k.shape)}")
        for t in (k_scale, v_scale):
            if t.dtype is not torch.float32 or tuple(t.shape) != (P, H, page):
                raise ValueError(f"cache scales must be float32 {(P, H, page)}, got {t.dtype} {tuple(t.shape)}")
        for t in (k, v, k_scale, v_scale):
            if not t.is_contiguous() or t.data_ptr() & 15:
                raise ValueError("cache tensors must be contiguous and 16-byte aligned")
            if t.device != k.device:
                raise ValueError(f"cache tensors lie on {t.device} and {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = P, H, page, D
        self.device, self._index = k.device, k.get_device()
        self._c = _CCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, H, page, D,
                          kinds[k.dtype])
        self._p = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, num_pages, page_size, kv_heads, head_dim, kind="int8", device="cuda"):
        """A cache of zeros; ``kind`` is "int8" or "fp8" (e4m3)."""
        torch = _torch()
        if kind not in ("int8", "fp8"):
            raise ValueError(f"kind must be 'int8' or 'fp8', got {kind!r}")
        shape = (int(num_pages), int(kv_heads), int(page_size))
        pages = [torch.zeros((*shape, int(head_dim)), dtype=torch.int8, device=device) for _ in range(2)]
        if kind == "fp8":
            pages = [p.view(torch.float8_e4m3fn) for p in pages]
        return cls(*pages, *(torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)))


def kv_write(cache, k, v, slots):
    """Quantize new tokens' keys and values into the cache.

    ``k``, ``v``: ``[T, kv_heads, head_dim]`` of one type (views of a wider
    projection are read in place); ``slots``: int32 ``[T]``, a token's page
    times the page size plus its place in the page.  A slot outside the cache
    (-1, say) skips its token; no slot may occur twice in a call.

    INT8: the scale is max|x| / 127 in fp32, the value the whole number nearest
    to x / scale, ties to even.  e4m3: the scale is the smallest power of two
    that brings the row within 448.  A row that holds an infinity or NaN reads
    back as NaN."""
    torch = _torch()
    shape = (k.shape[0] if k.dim() else 0, cache.kv_heads, cache.head_dim)
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"k and v must be [T, {cache.kv_heads}, {cache.head_dim}], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    dt = _type(k, "k")
    if v.dtype is not k.dtype:
        raise ValueError(f"k and v must have one type, got {k.dtype} and {v.dtype}")
    _ints(slots, (shape[0],), "slots")
    _same_device(cache._index, k, v, slots)
    if shape[0] == 0:
        return
    if cache._index != _current():
        with torch.cuda.device(cache.device):
            return kv_write(cache, k, v, slots)
    k, v = _rows(k, "k"), _rows(v, "v")
    ks, vs = k.stride(), v.stride()
    rc = hb._lib.i4_kv_write_dev(cache._p, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], shape[0], dt,
                                 slots.data_ptr(), hb._torch_stream(k))
    if rc:
        hb._check_rc(rc, "i4_kv_write_dev")


def kv_read(cache, slots, dtype):
    """The tokens of int32 ``slots`` [T] as (k, v), each ``[T, kv_heads,
    head_dim]`` of ``dtype``: the fp32 product of value and scale, rounded to the
    type.  Zeros where a slot is outside the cache."""
    torch = _torch()
    if dtype not in _dtypes:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    T = slots.shape[0] if slots.dim() else 0
    _ints(slots, (T,), "slots")
    _same_device(cache._index, slots)
    if cache._index != _current():
        with torch.cuda.device(cache.device):
            return kv_read(cache, slots, dtype)
    shape = (T, cache.kv_heads, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.device)
    v = torch.empty(shape, dtype=dtype, device=cache.device)
    if T:
        rc = hb._lib.i4_kv_read_dev(cache._p, k.data_ptr(), v.data_ptr(), T, _dtypes[dtype], slots.data_ptr(),
                                    hb._torch_stream(k))
        if rc:
            hb._check_rc(rc, "i4_kv_read_dev")
    return k, v


def _output(out, like, shape, what):
    torch = hb._torch
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    st = out.stride()
    if out.dtype is not like.dtype or out.shape != shape or out.device != like.device:
        raise ValueError(f"{what} must be {like.dtype} {shape} on {like.device}, got {out.dtype} {tuple(out.shape)} on "
                         f"{out.device}")
    if st[2] != 1 or (st[0] | st[1]) & 3 or out.data_ptr() & 15 or st[1] < shape[2] or st[0] < shape[1] * st[1]:
        raise ValueError(f"{what} needs a contiguous last dimension, strides of multiples of four elements, rows that "
                         f"do not overlap and 16-byte alignment, got strides {st}")
    return out


def _span(t):
    n = sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _no_overlap(out, t, what):
    """`out` is apart from `t`, or the same rows at the same places."""
    a, b = _span(out), _span(t)
    if a[0] < b[1] and b[0] < a[1] and not (a == b and out.stride() == t.stride()):
        raise ValueError(f"out overlaps {what}: it may be {what} itself, or apart from it")


def _apart(out, t, what):
    """An output shares no memory with an input of a call that reads it late."""
    a, b = _span(out), _span(t)
    if a[0] < b[1] and b[0] < a[1]:
        raise ValueError(f"{what} overlaps an input")


def paged_attention(q, cache, block_table, kv_lens, cu_q=None, scale=None, out=None):
    """Causal attention of new tokens over the cache; ``[T, heads, head_dim]``
    of q's type.

    ``q``: ``[T, heads, head_dim]``, the sequences' new tokens one after another
    (heads a multiple of the cache's; query head i reads key-value head i //
    (heads // kv_heads)).  ``block_table``: int32 ``[B, columns]``, each
    sequence's pages in order.  ``kv_lens``: int32 ``[B]``, each sequence's keys
    in the cache, its new tokens' included (``kv_write`` comes first).
    ``cu_q``: int32 ``[B + 1]``, where each sequence's new tokens begin and the
    last one's end; None: one token a sequence, T = B.  New token i of n sees
    the keys up to kv_len - n + i.  ``scale`` > 0 is the softmax scale
    (head_dim ** -0.5).

    A row that sees no key is zero; keys in pages outside the cache are not seen; a
    kv_len past the table's columns counts as what the table has room for; rows
    outside every sequence are not written.  ``out`` may be given: q itself, or
    apart from it.

    Sums and softmax statistics are fp32 and the cache's values enter the
    products exactly.  fp32 queries and their probabilities keep 22 bits; with
    bf16, and with fp16 in chunks of 512 keys and more, the probabilities are
    rounded to fp16's 11 bits.  Elements of a query are kept down to 2^-38 of its
    largest, a key's part in the sum down to 2^-30 of the largest value that the
    row sees among the 32 or 64 keys next to it.  NaN in a query or in a seen key
    spoils its row, as do scores past fp32's range (keys above some 1e31).

    The host does not read the lengths: how keys are split, whether long chunks'
    keys are unpacked first (up to 4 GiB of workspace) and how many partial sums
    there are (up to 1 GiB) go by the table's columns.  Where the columns that the
    batch needs are known, ``block_table[:, :n]`` is enough, and faster: a
    4096-token prompt takes 190 us so, 310 with a table of 131072 keys."""
    torch = _torch()
    T, heads, D = q.shape if q.dim() == 3 else (0, 0, 0)
    if D != cache.head_dim or heads % cache.kv_heads or not heads:
        raise ValueError(f"q must be [T, a multiple of {cache.kv_heads} heads, {cache.head_dim}], got {tuple(q.shape)}")
    dt = _type(q, "q")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, columns], got {tuple(block_table.shape)}")
    B, cols = block_table.shape
    _ints(block_table, (B, cols), "block_table")
    _ints(kv_lens, (B,), "kv_lens")
    if cu_q is not None:
        _ints(cu_q, (B + 1,), "cu_q")
    elif T != B:
        raise ValueError(f"{T} tokens in {B} sequences: cu_q says where each begins")
    if scale is None:
        scale = D ** -0.5
    elif not 0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    _same_device(cache._index, q, block_table, kv_lens, cu_q, out)
    given = out is not None
    out = _output(out, q, (T, heads, D), "out")
    if T == 0 or B == 0:
        return out
    if cache._index != _current():
        with torch.cuda.device(cache.device):
            return paged_attention(q, cache, block_table, kv_lens, cu_q, scale, out)
    q = _rows(q, "q")
    if given:
        _no_overlap(out, q, "q")
    lib = hb._lib
    work, n = _workspace((cache.kv_heads, cache.page_size, D, T, B, heads, dt, cols, cu_q is not None), "paged", q.device)
    qs, os = q.stride(), out.stride()
    rc = lib.i4_paged_attention_dev(
        cache._p, q.data_ptr(), qs[0], qs[1], T, heads, dt, block_table.data_ptr(), block_table.stride(0), cols,
        kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), B, scale, out.data_ptr(), os[0], os[1],
        None if work is None else work.data_ptr(), n, hb._torch_stream(q))
    if rc:
        hb._check_rc(rc, "i4_paged_attention_dev")
    return out


def _gates(t, shape, what):
    torch = hb._torch
    if t.shape != shape or t.dtype not in _dtypes:
        raise ValueError(f"{what} must be {shape} of float32, bfloat16 or float16, got {t.dtype} {tuple(t.shape)}")
    if t.dtype is not torch.float32 or (shape[1] > 1 and t.stride(1) != 1):
        t = t.to(torch.float32).contiguous()
    return t


def _state(t, shape, device, what):
    torch = hb._torch
    if t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous() or t.data_ptr() & 15:
        raise ValueError(f"{what} must be contiguous, 16-byte aligned float32 {shape}, got {t.dtype} {tuple(t.shape)} "
                         f"(strides {t.stride()})")


def gated_linear_attention(q, k, v, g, beta=None, state=None, cu_seqlens=None, scale=None, out=None, state_out=None):
    """Linear attention with a decay for each head and token, by the delta rule
    where ``beta`` is given; ``(o, state)``.

    For each value head, with the q and k of key head i // (v_heads //
    k_heads)::

        S_t = exp(g_t) S_{t-1} + k_t u_t^T          o_t = scale S_t^T q_t
        u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t)      (v_t without beta)

    ``q``, ``k``: ``[T, k_heads, k_dim]``; ``v``: ``[T, v_heads, v_dim]``, of one
    type (views of a wider projection are read in place).  ``g``, ``beta``:
    ``[T, v_heads]``; g is the decay's logarithm, at most 0 (-inf drops a
    finite state).  ``state``: fp32 ``[B, v_heads, k_dim, v_dim]``, what each sequence
    starts from (None: zeros).  ``cu_seqlens``: int32 ``[B + 1]``, where each
    sequence's tokens begin and the last one's end; None: one token a sequence,
    B = T.  A sequence without tokens keeps its state; rows outside every
    sequence are not written.  k_dim is 64 or 128, v_dim a multiple of 16 up to
    1024; ``scale`` is k_dim ** -0.5.

    The new state goes to ``state_out`` (``state`` itself, or apart from it) or
    to a new tensor.  State and sums are fp32; the products of prompts keep 22
    bits of every operand, of q and k down to 2^-28 of the largest in their chunk
    of 64 tokens and head, of v and the state down to 2^-37 of the largest in their
    column there.  With bf16 the state and u have 11 bits in the products that make
    rows of o, three more than those keep.  With beta, those bounds are for what the
    delta rule is stable for, beta |k|^2 up to 2: past that u grows from token to token,
    and a chunk's earlier rows lose bits to its largest u.

    A NaN in k, v, g or beta reaches its token's row and those after it (from v: in its
    column), one in q its own row; no earlier ones.  Sequences of more than 16
    tokens go in chunks of 64, where an infinity does as NaN does; their operands
    take up to 1 GiB of workspace, which longer prompts go through in segments."""
    torch = _torch()
    if q.dim() != 3 or v.dim() != 3 or k.shape != q.shape or v.shape[0] != q.shape[0]:
        raise ValueError(f"q and k must be [T, k_heads, k_dim] and v [T, v_heads, v_dim], got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    T, Hk, Dk = q.shape
    _, Hv, Dv = v.shape
    dt = _type(q, "q")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if not Hk or not Hv or Hv % Hk or Dk not in (64, 128) or Dv % 16 or not 16 <= Dv <= 1024:
        raise ValueError(f"needs v_heads in multiples of k_heads, k_dim 64 or 128 and v_dim a multiple of 16 up to 1024, "
                         f"got {Hv} of {Dv} and {Hk} of {Dk}")
    g = _gates(g, (T, Hv), "g")
    if beta is not None:
        beta = _gates(beta, (T, Hv), "beta")
    if cu_seqlens is None:
        B = T
    else:
        B = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
        if B < 0:
            raise ValueError(f"cu_seqlens must be [B + 1], got {tuple(cu_seqlens.shape)}")
        _ints(cu_seqlens, (B + 1,), "cu_seqlens")
    shape = (B, Hv, Dk, Dv)
    if state is not None:
        _state(state, shape, q.device, "state")
    if state_out is not None:
        _state(state_out, shape, q.device, "state_out")
    if scale is None:
        scale = Dk ** -0.5
    elif not -1e30 < scale < 1e30:
        raise ValueError(f"scale must be finite, got {scale}")
    index = q.get_device()
    _same_device(index, k, v, g, beta, state, cu_seqlens, state_out, out)
    given = out is not None
    out = _output(out, q, (T, Hv, Dv), "out")
    state_given = state_out is not None
    if not state_given:
        state_out = torch.empty(shape, dtype=torch.float32, device=q.device)
    elif state is not None:
        _no_overlap(state_out, state, "state")
    if B == 0:
        return out, state_out
    if index != _current():
        with torch.cuda.device(q.device):
            return gated_linear_attention(q, k, v, g, beta, state, cu_seqlens, scale, out, state_out)
    q, k, v = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    if given:
        for t in (q, k, v, g, beta, state, state_out):
            if t is not None:
                _apart(out, t, "out")
    if state_given:
        for t in (q, k, v, g, beta):
            if t is not None:
                _apart(state_out, t, "state_out")
    lib = hb._lib
    if cu_seqlens is None:
        work, n = None, 0
    else:
        work, n = _workspace((T, B, Hk, Hv, Dk, Dv, dt, True, beta is not None),
                             "gla", q.device)
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    rc = lib.i4_gated_linear_attention_dev(
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], g.data_ptr(), g.stride(0),
        None if beta is None else beta.data_ptr(), 0 if beta is None else beta.stride(0), T, Hk, Hv, Dk, Dv, dt,
        None if cu_seqlens is None else cu_seqlens.data_ptr(), B, scale, None if state is None else state.data_ptr(),
        state_out.data_ptr(), out.data_ptr(), os[0], os[1], None if work is None else work.data_ptr(), n,
        hb._torch_stream(q))
    if rc:
        hb._check_rc(rc, "i4_gated_linear_attention_dev")
    return out, state_out
