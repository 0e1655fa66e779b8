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
- ``Rotary`` and ``rotary``: positions of queries and keys ahead of the cache
  (the decoder's rope, kernel/qwen35_decoder.cpp:218-428).
- ``PageTable``: which pages sequences hold, and new tokens' slots and positions.

Tensors are fp32, bf16 or fp16 on one gfx950 GPU.  Calls are asynchronous on
the current stream, own no memory between calls (a workspace comes from
torch's allocator) and can be captured into graphs.  Shapes, types and strides
are checked here and raise ``ValueError``; what lies on the GPU (lengths,
offsets, page and slot numbers) is checked by the kernels, which skip what is
out of range.  Outputs carry no gradient.  There is no CPU fallback.
"""
import ctypes
import math

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
        n = getattr(hb._lib, _queries[kind])(*shape)
        if n < 0:
            raise ValueError(hb.last_error())
        if len(_needs) >= 4096:
            _needs.clear()
        _needs[key] = n
    return (hb._torch.empty((n,), dtype=hb._torch.uint8, device=device) if n else None), n


_needs = {}
_queries = {"paged": "i4_paged_attention_workspace", "gla": "i4_gated_linear_attention_workspace",
            "tree": "i4_tree_attention_workspace", "verify": "i4_verify_workspace"}


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
        self._geometry, self._k = (P, H, page, D, self._index), k.data_ptr()
        self._c = _CCache(self._k, v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, H, page, D,
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


class Rotary:
    """The angles of ``rotary``: of pair i of a head's first ``dim`` values,
    position times f_i radians, f_i = base ** (-2 i / dim).

    ``layout``: "half" (values i and i + dim / 2 are a pair) or "interleaved" (2 i
    and 2 i + 1).  ``scaling`` for contexts ``factor`` times as long:

    - "linear": all f_i divided by the factor;
    - "base": the base times factor ** (dim / (dim - 2)), so that the slowest f_i
      is divided by the factor and the fastest stays;
    - "parts": a pair that turns more than ``fast`` times in the ``original``
      context keeps its f_i, one that turns less than ``slow`` times has it divided,
      those in between are mixed linearly in the turns; sine and cosine are
      multiplied by 0.1 ln(factor) + 1 (or ``amplitude``).

    ``freqs``: f_i themselves (dim / 2 numbers), in place of all that, for other
    scalings: one that goes from kept to divided along the pairs' numbers i, say,
    where "parts" goes by their turns.  They are kept in 64 bits on ``device``, as
    quarter turns."""

    def __init__(self, dim, base=10000.0, layout="half", scaling=None, factor=1.0, original=None, slow=1.0, fast=32.0,
                 amplitude=None, freqs=None, device="cuda"):
        torch = _torch()
        if dim < 2 or dim % 2 or dim > 4096:
            raise ValueError(f"dim must be even, from 2 to 4096, got {dim}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if scaling not in (None, "linear", "base", "parts"):
            raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
        if not 0 < base < math.inf or not 0 < factor < math.inf:
            raise ValueError(f"base and factor must be positive and finite, got {base} and {factor}")
        if freqs is not None:
            f = [float(x) for x in freqs]
            if len(f) != dim // 2 or scaling is not None:
                raise ValueError(f"freqs must be {dim // 2} numbers, without scaling, got {len(f)}")
        else:
            if scaling == "base" and dim > 2:
                base = base * factor ** (dim / (dim - 2))
            f = [base ** (-2 * i / dim) for i in range(dim // 2)]
            if scaling == "linear":
                f = [x / factor for x in f]
            elif scaling == "parts":
                if not original or original < 1 or not 0 <= slow < fast:
                    raise ValueError(f"'parts' needs the original context and slow < fast, got {original}, {slow}, {fast}")
                for i, x in enumerate(f):
                    keep = min(max((original * x / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0)
                    f[i] = x * (keep + (1 - keep) / factor)
                if amplitude is None:
                    amplitude = 0.1 * math.log(factor) + 1
        self.dim, self.layout, self.amplitude = dim, layout, 1.0 if amplitude is None else float(amplitude)
        if not all(math.isfinite(x) for x in (*f, self.amplitude)):
            raise ValueError("freqs and amplitude must be finite")
        self._turns = torch.tensor([x * (2 / math.pi) for x in f], dtype=torch.float64, device=device)
        self.device, self._index = self._turns.device, self._turns.get_device()
        self._p, self._inter = self._turns.data_ptr(), int(layout == "interleaved")


def _heads(t, T, D, what):
    """`t` [T, heads, D] with a contiguous last dimension: itself, or a copy."""
    if t.dim() != 3 or t.shape[0] != T or t.shape[2] != D:
        raise ValueError(f"{what} must be [{T}, heads, {D}], got {tuple(t.shape)}")
    return t if t.stride(2) == 1 else t.contiguous()


def _turned(out, like, what):
    if out is None:
        return like.new_empty(like.shape)
    T, H, D = like.shape
    st = out.stride()
    if out.dtype is not like.dtype or out.shape != like.shape or out.device != like.device:
        raise ValueError(f"{what} must be {like.dtype} {tuple(like.shape)} on {like.device}, got {out.dtype} "
                         f"{tuple(out.shape)} on {out.device}")
    if st[2] != 1 or (H > 1 and st[1] < D) or (T > 1 and st[0] < (H - 1) * st[1] + D):
        raise ValueError(f"{what} needs a contiguous last dimension and rows that do not overlap, got strides {st}")
    return out


def _same_rows(a, b):
    """a and b, of one shape and type, are the same rows at the same places."""
    return a.data_ptr() == b.data_ptr() and all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


def _disjoint(a, b):
    """No row of a lies on one of b: they are apart, or other columns of one projection, of
    its tokens or of its heads."""
    x, y = _span(a), _span(b)
    if x[0] >= y[1] or y[0] >= x[1]:
        return True
    if a.dtype is not b.dtype:
        return False
    size = a.element_size()
    for t, d in ((a, 0), (b, 0), (a, 1), (b, 1)):
        step = t.stride(d) * size
        if t.shape[d] < 2 or step == 0:
            continue
        # The bytes of each, from the first row's on, modulo the step: a dimension that goes on by
        # whole steps adds none.
        wide = [sum((t.shape[i] - 1) * t.stride(i) * size for i in (0, 1) if t.stride(i) * size % step) + t.shape[2] * size
                for t in (a, b)]
        apart = (y[0] - x[0]) % step
        if wide[0] <= apart and apart + wide[1] <= step:
            return True
    return False


def rotary(rope, q, k, positions, out=None):
    """Rotary positions of queries and keys; ``(q, k)``, turned.

    ``q``: ``[T, heads, head_dim]``; ``k``: ``[T, kv_heads, head_dim]`` of q's type,
    or None; ``positions``: int32 ``[T]``, each token's (``PageTable.extend`` gives
    them).  The first ``rope.dim`` values of a head are turned, in fp32 with angles
    from 64 bits, at whatever position; the others are copied.

    Views are read in place.  ``out``: (q, k) to write to, each the input itself
    or apart from both inputs (other columns of one projection, or of its heads, are).
    Where all are the inputs themselves only what is turned is written."""
    torch = _torch()
    T, _, D = q.shape if q.dim() == 3 else (0, 0, 0)
    dt = _type(q, "q")
    q = _heads(q, T, D, "q")
    if D % 2 or D < rope.dim or D > 4096:
        raise ValueError(f"head_dim must be even, from the rotary's {rope.dim} to 4096, got {D} (q: {tuple(q.shape)})")
    if k is not None:
        k = _heads(k, T, D, "k")
        if k.dtype is not q.dtype:
            raise ValueError(f"q and k must have one type, got {q.dtype} and {k.dtype}")
    _ints(positions, (T,), "positions")
    _same_device(rope._index, q, k, positions)
    if out is None:
        qo, ko = _turned(None, q, "q"), None if k is None else _turned(None, k, "k")
    else:
        qo, ko = out
        if qo is None or (ko is None) != (k is None):
            raise ValueError("out must be (q, k), with None where k is None")
        qo = _turned(qo, q, "out's q")
        ko = None if k is None else _turned(ko, k, "out's k")
        if T:
            for o, own, other, there in ((qo, q, k, ko), (ko, k, q, qo)):
                if o is None:
                    continue
                if not _same_rows(o, own) and not _disjoint(o, own):
                    raise ValueError("out overlaps its input: it may be the input itself, or apart from it")
                if other is not None and not (_disjoint(o, other) and _disjoint(o, there)):
                    raise ValueError("out's q and k lie on one another, or on the other's input")
    if T == 0:
        return qo, ko
    if rope._index != _current():
        with torch.cuda.device(rope.device):
            return rotary(rope, q, k, positions, (qo, ko))
    qs, os = q.stride(), qo.stride()
    if k is None:
        kp, ks, kn, kop, kos = None, (0, 0), 0, None, (0, 0)
    else:
        kp, ks, kn, kop, kos = k.data_ptr(), k.stride(), k.shape[1], ko.data_ptr(), ko.stride()
    rc = hb._lib.i4_rotary_dev(q.data_ptr(), qs[0], qs[1], q.shape[1], kp, ks[0], ks[1], kn, T, D, rope.dim, rope._inter,
                               dt, positions.data_ptr(), rope._p, rope.amplitude, qo.data_ptr(), os[0], os[1], kop,
                               kos[0], kos[1], hb._torch_stream(q))
    if rc:
        hb._check_rc(rc, "i4_rotary_dev")
    return qo, ko


class PageTable:
    """Which pages of a cache a batch's sequences hold, on the GPU.

    ``table``: int32 ``[B, columns]``, each sequence's pages in order (the
    ``block_table`` of attention), of which it holds the first ``held`` (int32
    ``[B]``); ``free``: int32 ``[pages]``, the first ``count`` (int32 ``[1]``) of which
    are the free pages, a stack.  The tensors are kept as given and changed in
    place, in the order of the stream's calls; the host reads none of them."""

    def __init__(self, table, held, free, count, page_size):
        torch = _torch()
        if page_size & (page_size - 1) or not 16 <= page_size <= 1024:
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if table.dim() != 2 or free.dim() != 1 or not free.shape[0]:
            raise ValueError(f"table must be [B, columns] and free [pages], got {tuple(table.shape)} and "
                             f"{tuple(free.shape)}")
        B, cols = table.shape
        if B > 1 << 20 or B * cols >= 1 << 31 or cols * page_size > 1 << 30 or free.shape[0] * page_size >= 1 << 31:
            raise ValueError(f"a table has up to 2^20 sequences, fewer than 2^31 entries and up to 2^30 keys a sequence, a "
                             f"cache fewer than 2^31 slots, got {B}, {cols} columns and {free.shape[0]} pages of {page_size}")
        for t, shape, what in ((table, (B, cols), "table"), (held, (B,), "held"), (free, tuple(free.shape), "free"),
                               (count, (1,), "count")):
            if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous int32 {shape}, got {t.dtype} {tuple(t.shape)}")
            if t.device != table.device:
                raise ValueError(f"the page table's tensors lie on {t.device} and {table.device}")
        self.table, self.held, self.free, self.count, self.page_size = table, held, free, count, page_size
        self.device, self._index = table.device, table.get_device()
        self._args = (table.data_ptr(), held.data_ptr(), free.data_ptr(), count.data_ptr(), free.shape[0], page_size, B,
                      cols)

    @classmethod
    def empty(cls, num_pages, page_size, batch, columns, device="cuda"):
        """A table of ``batch`` sequences that hold nothing; all pages are free."""
        torch = _torch()
        new = lambda *shape, **kw: torch.full(shape, dtype=torch.int32, device=device, **kw)  # noqa: E731
        free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(new(batch, columns, fill_value=-1), new(batch, fill_value=0), free, new(1, fill_value=num_pages),
                   page_size)

    def extend(self, lens, cu=None, tokens=None, parents=None):
        """Room for new tokens; ``(slots, positions, kv_lens)``.

        ``lens``: int32 ``[B]``, each sequence's tokens in the cache.  ``cu``: int32
        ``[B + 1]``, where each sequence's new tokens begin and the last one's end, of
        ``tokens`` in all; None: one each.  ``parents``: int32 ``[tokens]``, the new
        tokens being trees (``drafts.tree_attention``).

        Pages come off the stack for the sequences in order.  ``slots`` are
        ``kv_write``'s, ``positions`` the tokens' own: lens + the token's number, or
        its depth in the tree; ``kv_lens`` the lengths with the new tokens.  Where the
        pages do not suffice, that sequence and every later one that needs pages get
        none; those, sequences past the table's columns or of a negative length, and
        trees past 1024 nodes, have a kv_len and slots of -1: no call writes or sees
        anything of them, and ``drafts.verify`` and ``kv_compact`` take kv_lens and lens, so
        that they get no token and keep their length and pages for a later step.  Tokens outside every sequence have slot -1."""
        torch = _torch()
        B = self._args[6]
        _ints(lens, (B,), "lens")
        if cu is None:
            T = B
            if tokens not in (None, B):
                raise ValueError(f"{tokens} tokens in {B} sequences: cu says where each begins")
        else:
            _ints(cu, (B + 1,), "cu")
            if tokens is None and parents is not None:
                tokens = parents.numel()
            if tokens is None or tokens < 0:
                raise ValueError(f"with cu, tokens says how many there are in all, got {tokens}")
            T = int(tokens)
        if parents is not None:
            _ints(parents, (T,), "parents")
        _same_device(self._index, lens, cu, parents)
        if self._index != _current():
            with torch.cuda.device(self.device):
                return self.extend(lens, cu, T, parents)
        # One allocation: the host part is most of a small call.
        new = lens.new_empty((2 * T + B,))
        p = new.data_ptr()
        rc = hb._lib.i4_pages_extend_dev(*self._args, lens.data_ptr(), None if cu is None else cu.data_ptr(), T,
                                         None if parents is None else parents.data_ptr(), p, p + 4 * T, p + 8 * T,
                                         hb._torch_stream(lens))
        if rc:
            hb._check_rc(rc, "i4_pages_extend_dev")
        return new.split((T, T, B))

    def trim(self, lens):
        """Pages past ``lens`` (int32 ``[B]``) tokens of each sequence go back to the
        stack: 0 gives all of a sequence's, a negative length none.  Table entries that
        go become -1."""
        torch = _torch()
        _ints(lens, (self._args[6],), "lens")
        _same_device(self._index, lens)
        if self._index != _current():
            with torch.cuda.device(self.device):
                return self.trim(lens)
        rc = hb._lib.i4_pages_trim_dev(*self._args, lens.data_ptr(), hb._torch_stream(lens))
        if rc:
            hb._check_rc(rc, "i4_pages_trim_dev")


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
