"""What rotary positions, page tables and the calls on drafted tokens refuse, on
the CPU: the Python layer's checks and the C entry points' own, all before any
GPU call."""
import ctypes

import pytest
import torch

from breeze_amd import attention as att
from breeze_amd import drafts
from breeze_amd import hip_backend as hb

I32 = torch.int32


def _ints(*shape):
    return torch.zeros(shape, dtype=I32)


@pytest.fixture
def cache():
    return att.KVCache.empty(3, 16, 2, 64, device="cpu")


def _raises(f, calls, **known):
    for args, kw in calls:
        with pytest.raises(ValueError):
            f(*args, **dict(known, **kw))


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(dim=5000), dict(layout="other"), dict(scaling="more"),
                                dict(base=0.0), dict(base=float("inf")), dict(factor=0.0), dict(factor=float("nan")),
                                dict(scaling="parts"), dict(scaling="parts", original=100, slow=40.0),
                                dict(freqs=[1.0]), dict(freqs=[1.0] * 32, scaling="linear"),
                                dict(freqs=[float("nan")] * 32), dict(amplitude=float("nan")),
                                dict(amplitude=float("inf"))])
def test_rotary_objects(kw):
    with pytest.raises(ValueError):
        att.Rotary(**dict(dict(dim=64, device="cpu"), **kw))


def test_rotary():
    rope = att.Rotary(64, device="cpu")
    q, k, at = torch.zeros((4, 6, 128)), torch.zeros((4, 2, 128)), _ints(4)
    with pytest.raises(ValueError, match="GPU"):
        att.rotary(rope, q, k, at)
    _raises(att.rotary, [((rope, q[0], k, at), {}), ((rope, q, k[:3], at), {}), ((rope, q, k[:, :, :64], at), {}),
                         ((rope, q.double(), k.double(), at), {}), ((rope, q, k.half(), at), {}),
                         ((rope, q, k, at.long()), {}), ((rope, q, k, at[:3]), {}), ((rope, q, k, at[:, None]), {}),
                         ((rope, q[..., :32], None, at), {}), ((rope, q[..., :65], None, at), {})])


def test_rotary_outputs():
    q = torch.zeros((4, 6, 128))
    assert att._turned(q, q, "out") is q
    for bad in (q.half(), q[:3], torch.zeros((4, 6, 256))[..., ::2], torch.zeros((1, 6, 128)).expand(4, 6, 128),
                torch.zeros((6, 4, 128)).transpose(0, 1), torch.zeros((4, 1, 128)).expand(4, 6, 128)):
        with pytest.raises(ValueError):
            att._turned(bad, q, "out")
    wide = torch.zeros((4, 9 * 128))
    a, b = wide[:, :768].view(4, 6, 128), wide[:, 768:1024].view(4, 2, 128)
    c = wide[:, 640:896].view(4, 2, 128)
    assert att._disjoint(a, b) and att._disjoint(b, a) and att._disjoint(a, torch.zeros((4, 6, 128)))
    assert not att._disjoint(a, c) and not att._disjoint(c, b) and not att._disjoint(a, a)
    # Columns that wrap round into the next token's, another step, no step.
    late = wide.view(-1)[1100:1100 + 3 * 1152].view(3, 1152)[:, :256].view(3, 2, 128)
    assert not att._disjoint(a[:3], late) and att._disjoint(b[:3], late[..., :52])
    assert not att._disjoint(a, wide.view(-1)[:4 * 256].view(4, 2, 128))


def test_page_tables():
    def make(B=2, cols=3, P=5, page=16, **kw):
        t = dict(table=_ints(B, cols), held=_ints(B), free=_ints(P), count=_ints(1))
        t.update(kw)
        return att.PageTable(*t.values(), page)

    make()
    for kw in (dict(page=8), dict(page=24), dict(page=2048), dict(P=0), dict(table=_ints(6)), dict(table=_ints(2, 3).long()),
               dict(held=_ints(3)), dict(count=_ints(2)), dict(count=torch.zeros(1)), dict(free=_ints(5, 1)),
               dict(table=_ints(3, 2).t()), dict(free=_ints(10)[::2])):
        with pytest.raises(ValueError):
            make(**kw)
    pt = att.PageTable.empty(5, 16, 2, 3, device="cpu")
    assert pt.free.tolist() == [4, 3, 2, 1, 0] and pt.count.tolist() == [5] and pt.table.eq(-1).all()
    with pytest.raises(ValueError, match="GPU"):
        pt.extend(_ints(2))
    with pytest.raises(ValueError, match="GPU"):
        pt.trim(_ints(2))
    _raises(pt.extend, [((_ints(3),), {}), ((_ints(2).long(),), {}), ((_ints(2),), dict(tokens=3)),
                        ((_ints(2), _ints(3)), {}), ((_ints(2), _ints(2), 4), {}), ((_ints(2), _ints(3), -1), {}),
                        ((_ints(2), _ints(3).long(), 4), {}), ((_ints(2), _ints(3), 4, _ints(5)), {}),
                        ((_ints(2), _ints(3), 4, _ints(4).long()), {}),
                        ((_ints(2), _ints(3), None, _ints(1)[0]), {})])
    _raises(pt.trim, [((_ints(3),), {}), ((torch.zeros(2),), {})])


def test_tree_attention(cache):
    q, table, lens, up = torch.zeros((4, 6, 64)), _ints(4, 2), _ints(4), _ints(4)
    cu = torch.arange(5, dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        drafts.tree_attention(q, cache, table, lens, up, cu)
    ok = (q, cache, table, lens, up, cu)
    swap = lambda i, x: tuple(x if j == i else y for j, y in enumerate(ok))  # noqa: E731
    _raises(drafts.tree_attention, [
        (swap(0, q[0]), {}), (swap(0, q[:, :5]), {}), (swap(0, q[:, :0]), {}), (swap(0, q[..., :32]), {}),
        (swap(0, q.double()), {}), (swap(0, q[:3]), {}), (swap(2, table[0]), {}), (swap(2, table.long()), {}),
        (swap(2, _ints(4, 4)[:, ::2]), {}), (swap(3, lens.long()), {}), (swap(3, lens[:3]), {}), (swap(4, up[:3]), {}),
        (swap(4, up.long()), {}), (swap(4, _ints(8)[::2]), {}), (swap(5, cu[:4]), {}), (swap(5, cu.long()), {}),
        ((q[:3], cache, table, lens, up[:3]), {}), (ok, dict(scale=0.0)), (ok, dict(scale=-1.0)),
        (ok, dict(scale=float("nan"))), (ok, dict(scale=float("inf"))), (ok, dict(out=q.half()))])


def test_verify():
    x, t, up, u, cu = torch.zeros((5, 40)), _ints(5), _ints(5), torch.zeros(5), torch.tensor([0, 2, 5], dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        drafts.verify(x, t, up, u, cu)
    ok = (x, t, up, u, cu)
    swap = lambda i, y: tuple(y if j == i else z for j, z in enumerate(ok))  # noqa: E731
    nan, inf = float("nan"), float("inf")
    _raises(drafts.verify, [
        (swap(0, x[0]), {}), (swap(0, x.double()), {}), (swap(0, x[:, :0]), {}),
        (swap(0, torch.zeros(1).expand(5, (1 << 21) + 1)), {}),
        (swap(1, t.long()), {}), (swap(1, t[:4]), {}), (swap(2, up[:4]), {}), (swap(2, None), {}), (swap(3, u.double()), {}),
        (swap(3, u[:4]), {}), (swap(3, torch.zeros(10)[::2]), {}), (swap(4, cu.long()), {}), (swap(4, cu[:0]), {}),
        (swap(4, cu[None]), {}), (ok, dict(temperature=-0.5)), (ok, dict(temperature=nan)), (ok, dict(temperature=inf)),
        (ok, dict(temperature=torch.zeros(3))), (ok, dict(temperature=torch.zeros(2).half())),
        (ok, dict(temperature=torch.zeros(4)[::2])), (ok, dict(draft=x.half())), (ok, dict(draft=x[:4])),
        (ok, dict(draft=x[:, :39]))])


def test_kv_compact(cache):
    table, lens, cu, path, counts = _ints(2, 2), _ints(2), torch.tensor([0, 2, 5], dtype=I32), _ints(5), _ints(2)
    with pytest.raises(ValueError, match="GPU"):
        drafts.kv_compact(cache, table, lens, cu, path, counts)
    other = att.KVCache.empty(4, 16, 2, 64, device="cpu")
    ok = ([cache, att.KVCache.empty(3, 16, 2, 64, device="cpu")], table, lens, cu, path, counts)
    with pytest.raises(ValueError, match="GPU"):
        drafts.kv_compact(*ok)
    for twice in (cache, att.KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale)):
        with pytest.raises(ValueError, match="twice"):
            drafts.kv_compact([cache, twice], *ok[1:])
    swap = lambda i, y: tuple(y if j == i else z for j, z in enumerate(ok))  # noqa: E731
    _raises(drafts.kv_compact, [
        (swap(0, []), {}), (swap(0, [cache, other]), {}), (swap(0, [cache] * 4097), {}), (swap(1, table[0]), {}),
        (swap(1, table.long()), {}), (swap(2, lens[:1]), {}), (swap(3, cu[:2]), {}), (swap(3, None), {}),
        (swap(4, path.long()), {}), (swap(4, path[None]), {}), (swap(5, counts[:1]), {}), (swap(5, counts.long()), {})])


def _c_cache(**kw):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, num_pages=2, kv_heads=2, page_size=16, head_dim=64, kind=0)
    d.update(kw)
    return att._CCache(*(d[f] for f, _ in att._CCache._fields_))


def test_c_rotary():
    def call(q=4096, qh=2, k=4096, kh=1, T=1, D=64, rot=64, dt=0, at=4096, f=4096, qo=4096, ko=4096):
        return hb._lib.i4_rotary_dev(q, 128, 64, qh, k, 64, 64, kh, T, D, rot, 0, dt, at, f, 1.0, qo, 128, 64, ko, 64, 64,
                                     None)

    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(at=None), dict(f=None), dict(T=-1),
               dict(T=1 << 24), dict(D=63), dict(D=0), dict(D=5000, rot=64), dict(rot=0), dict(rot=66), dict(rot=7), dict(dt=3),
               dict(dt=-1), dict(qh=-1), dict(kh=70000)):
        assert call(**kw) == -2 and "rotary" in hb.last_error(), kw
    assert call(T=0) == 0 and call(qh=0, kh=0, q=None, k=None) == 0


def test_c_pages():
    def extend(table=4096, held=4096, free=4096, count=4096, P=9, page=16, B=2, cols=3, lens=4096, cu=4096, T=5, slots=4096,
               at=4096, kv=4096):
        return hb._lib.i4_pages_extend_dev(table, held, free, count, P, page, B, cols, lens, cu, T, None, slots, at, kv, None)

    for kw in (dict(table=None), dict(held=None), dict(free=None), dict(count=None), dict(lens=None), dict(slots=None),
               dict(at=None), dict(kv=None), dict(P=0), dict(P=1 << 28), dict(page=24), dict(page=8), dict(B=-1),
               dict(B=1 << 21), dict(cols=-1), dict(cols=1 << 27), dict(B=1 << 20, cols=1 << 12), dict(T=-1),
               dict(cu=None), dict(T=(1 << 30) + 1)):
        assert extend(**kw) == -2 and "pages_extend" in hb.last_error(), kw
    assert extend(B=0, T=0) == 0
    trim = hb._lib.i4_pages_trim_dev
    assert trim(4096, 4096, 4096, 4096, 9, 16, 2, 3, None, None) == -2 and "pages_trim" in hb.last_error()
    assert trim(4096, 4096, 4096, 4096, 9, 17, 2, 3, 4096, None) == -2
    assert trim(None, None, None, None, 9, 16, 0, 3, None, None) == 0


@pytest.mark.parametrize("kw", [dict(num_pages=0), dict(kv_heads=0), dict(kv_heads=4097), dict(page_size=24),
                                dict(head_dim=96), dict(kind=2), dict(k=None), dict(v_scale=None)])
def test_c_caches(kw):
    c = _c_cache(**kw)
    p = ctypes.addressof(c)
    rc = hb._lib.i4_tree_attention_dev(p, 4096, 128, 64, 1, 2, 0, 4096, 1, 1, 4096, None, 1, 4096, 0.1, 4096, 128, 64,
                                       None, 0, None)
    assert rc == -2 and "tree_attention" in hb.last_error()
    if kw != dict(kind=2):  # bytes are moved whatever they stand for
        several = (ctypes.c_void_p * 1)(p)
        assert hb._lib.i4_kv_compact_dev(several, 1, 4096, 1, 1, 4096, 4096, 3, 1, 4096, 4096, 8192, None) == -2
        assert "kv_compact" in hb.last_error()


def test_c_tree_attention():
    c = _c_cache()
    p = ctypes.addressof(c)

    def call(q=4096, T=4, heads=4, dt=0, table=4096, cols=1, lens=4096, cu=4096, B=2, up=4096, scale=0.1, out=4096):
        return hb._lib.i4_tree_attention_dev(p, q, 256, 64, T, heads, dt, table, cols, cols, lens, cu, B, up, scale, out,
                                             256, 64, None, 0, None)

    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(table=None), dict(up=None), dict(heads=3), dict(heads=0),
               dict(dt=3), dict(dt=-1), dict(cu=None), dict(T=-1), dict(B=-1), dict(cols=-1), dict(cols=1 << 28),
               dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e31), dict(T=1 << 26), dict(B=1 << 22)):
        assert call(**kw) == -2, kw
    assert call(T=0) == 0 and call(B=0) == 0
    assert call(cols=4096) == -4 and "workspace" in hb.last_error()
    need = hb._lib.i4_tree_attention_workspace
    assert need(2, 16, 64, 4, 2, 4, 0, 4096, 1) > 0 and need(2, 16, 64, 4, 2, 3, 0, 4096, 1) == -2
    assert need(2, 16, 64, 0, 2, 4, 0, 4096, 1) == 0
    assert need(2, 16, 64, (1 << 22) + 1, 2, 4, 0, 4096, 1) == -2 and need(2, 16, 64, 1 << 20, (1 << 19) + 1, 4, 0, 4096, 1) == -2


def test_workspaces_have_a_bound():
    """512 MiB of partial sums at most, whatever the table's columns and the nodes."""
    for D in (64, 128, 256):
        for H, heads in ((1, 1), (1, 128), (4, 24), (8, 32), (32, 32)):
            for T in (1, 2, 63, 1000, 8192, 65536):
                for B in (1, 2, 64, 1000):
                    for keys in (16, 1000, 4096, 131072, 1 << 22, 1 << 30):
                        for dtype in (0, 1):
                            if B <= T:
                                n = hb._lib.i4_tree_attention_workspace(H, 16, D, T, B, heads, dtype, -(-keys // 16), 1)
                                assert 0 <= n <= 512 << 20, (D, H, heads, T, B, keys, n)


def test_c_verify():
    def call(x=4096, T=4, V=100, dt=0, tokens=4096, u=4096, cu=4096, B=2, t=1.0, out=4096, path=4096, counts=4096, work=None,
             n=0):
        return hb._lib.i4_verify_dev(x, 100, T, V, dt, tokens, 4096, u, cu, B, None, t, None, 0, out, path, counts, work, n,
                                     None)

    for kw in (dict(x=None), dict(tokens=None), dict(u=None), dict(out=None), dict(path=None), dict(counts=None), dict(T=-1),
               dict(B=-1), dict(V=0), dict(V=(1 << 21) + 1), dict(dt=3), dict(cu=None), dict(t=-1.0), dict(t=float("nan")),
               dict(t=1e31), dict(T=1 << 23, V=4000), dict(T=1 << 23, B=(1 << 22) + 1)):
        assert call(**kw) == -2, kw
    assert call(B=0, T=0) == 0
    assert call() == -4 and "workspace" in hb.last_error()
    assert hb._lib.i4_verify_workspace(4, 100, 2, 1, 0) == 4 * (16 + 8)
    assert hb._lib.i4_verify_workspace(4, 0, 2, 1, 0) == -2


def test_c_compact():
    c = _c_cache()
    several = (ctypes.c_void_p * 2)(ctypes.addressof(c), ctypes.addressof(c))

    def call(caches=several, layers=2, table=4096, cols=1, kv=4096, cu=4096, T=4, B=2, path=4096, counts=4096, lens=8192):
        return hb._lib.i4_kv_compact_dev(caches, layers, table, cols, cols, kv, cu, T, B, path, counts, lens, None)

    for kw in (dict(caches=None), dict(layers=0), dict(layers=4097), dict(table=None), dict(kv=None), dict(path=None),
               dict(counts=None), dict(lens=None), dict(lens=4096), dict(cu=None), dict(T=-1), dict(B=-1), dict(cols=-1),
               dict(cols=1 << 28), dict(B=(1 << 22) + 1)):
        assert call(**kw) == -2 and "kv_compact" in hb.last_error(), kw
    d = _c_cache(num_pages=3)
    assert call(caches=(ctypes.c_void_p * 2)(ctypes.addressof(c), ctypes.addressof(d))) == -2
    assert call(caches=(ctypes.c_void_p * 2)(ctypes.addressof(c), None)) == -2
    assert call(B=0) == 0
