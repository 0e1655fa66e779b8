"""What the token mixers refuse, on the CPU: the Python layer's checks of
shapes, types and strides, and the C entry points' own, all before any GPU
call."""
import ctypes

import pytest
import torch

from breeze_amd import attention as att
from breeze_amd import hip_backend as hb


def _parts(P=3, H=2, page=16, D=64, dtype=torch.int8):
    return [torch.zeros((P, H, page, D), dtype=torch.int8).view(dtype) for _ in range(2)] + [
        torch.zeros((P, H, page)) for _ in range(2)]


@pytest.fixture
def cache():
    return att.KVCache(*_parts())


@pytest.mark.parametrize("kw", [dict(D=32), dict(D=96), dict(D=512), dict(page=8), dict(page=24), dict(page=2048),
                                dict(P=0), dict(H=0), dict(H=5000)])
def test_cache_shapes(kw):
    with pytest.raises(ValueError):
        att.KVCache(*_parts(**kw))


def test_cache_types_and_layout():
    k, v, ks, vs = _parts()
    for bad in ([k.float(), v, ks, vs], [k.view(torch.float8_e4m3fn), v, ks, vs], [k.view(torch.uint8)] * 2 + [ks, vs],
                [k, v[:2], ks, vs], [k[0], v[0], ks, vs], [k, v, ks.double(), vs], [k, v, ks, vs[:, :1]],
                [k.transpose(0, 1).contiguous().transpose(0, 1), v, ks, vs],
                [k, v, ks, torch.zeros(97)[1:].view(3, 2, 16)]):
        with pytest.raises(ValueError):
            att.KVCache(*bad)
    assert att.KVCache.empty(2, 32, 1, 128, "fp8", device="cpu").k.dtype is torch.float8_e4m3fn
    with pytest.raises(ValueError):
        att.KVCache.empty(2, 32, 1, 128, "int4", device="cpu")


def test_cache_writes_and_reads(cache):
    x, slots = torch.zeros((5, 2, 64)), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        att.kv_write(cache, x, x, slots)
    for k, v, s in ((x[:, :1], x, slots), (x, x[:4], slots), (x[:, :, :32], x, slots), (x.double(), x.double(), slots),
                    (x, x.half(), slots), (x, x, slots.long()), (x, x, slots[:4]), (x, x, slots[:, None]),
                    (x, x, torch.zeros(10, dtype=torch.int32)[::2]), (x[0], x[0], slots), (x.int(), x.int(), slots)):
        with pytest.raises(ValueError):
            att.kv_write(cache, k, v, s)
    with pytest.raises(ValueError, match="GPU"):
        att.kv_read(cache, slots, torch.float32)
    for s, dt in ((slots, torch.float64), (slots.long(), torch.float32), (slots[:, None], torch.float32)):
        with pytest.raises(ValueError):
            att.kv_read(cache, s, dt)


def test_paged_attention(cache):
    q, table, lens = torch.zeros((4, 6, 64)), torch.zeros((4, 2), dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    cu = torch.arange(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        att.paged_attention(q, cache, table, lens, cu)
    nan = float("nan")
    for args, kw in (((q[0], cache, table, lens), {}), ((q[:, :5], cache, table, lens), {}),
                     ((q[:, :0], cache, table, lens), {}), ((q[:, :, :32], cache, table, lens), {}),
                     ((q.double(), cache, table, lens), {}), ((q, cache, table[0], lens), {}),
                     ((q, cache, table.long(), lens), {}), ((q, cache, table, lens.long()), {}),
                     ((q, cache, table, lens[:3]), {}), ((q, cache, table, lens, cu[:4]), {}),
                     ((q, cache, table, lens, cu.long()), {}), ((q[:3], cache, table, lens), {}),
                     ((q, cache, torch.zeros((4, 4), dtype=torch.int32)[:, ::2], lens), {}),
                     ((q, cache, table, lens), dict(scale=0.0)), ((q, cache, table, lens), dict(scale=-1.0)),
                     ((q, cache, table, lens), dict(scale=nan)), ((q, cache, table, lens), dict(scale=float("inf")))):
        with pytest.raises(ValueError):
            att.paged_attention(*args, **kw)


def test_gated_linear_attention():
    q, v = torch.zeros((4, 2, 64)), torch.zeros((4, 4, 32))
    g, s, cu = torch.zeros((4, 4)), torch.zeros((4, 4, 64, 32)), torch.arange(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        att.gated_linear_attention(q, q, v, g, g, s, cu)
    inf = float("inf")
    for args, kw in (((q, q[:3], v, g), {}), ((q, q, v[:3], g), {}), ((q[0], q[0], v, g), {}),
                     ((q, q, v[:, :3], g[:, :3]), {}), ((q[:, :, :32], q[:, :, :32], v, g), {}),
                     ((q, q, v[:, :, :24], g), {}), ((q, q, v[:, :, :0], g), {}), ((q, q.half(), v, g), {}),
                     ((q.double(), q.double(), v.double(), g), {}), ((q, q, v, g[:, :3]), {}),
                     ((q, q, v, g.int()), {}), ((q, q, v, g, g[:3]), {}), ((q, q, v, g, g, s[:3]), {}),
                     ((q, q, v, g, g, s.half()), {}), ((q, q, v, g, g, s.transpose(2, 3)), {}),
                     ((q, q, v, g, g, s, cu[:0]), {}), ((q, q, v, g, g, s, cu.long()), {}),
                     ((q, q, v, g, g, s, cu[:, None]), {}), ((q, q, v, g, g, s, cu), dict(scale=inf)),
                     ((q, q, v, g, g, s, cu), dict(state_out=s[:3])), ((q, q, v, g, g, s, cu), dict(state_out=s.half()))):
        with pytest.raises(ValueError):
            att.gated_linear_attention(*args, **kw)


def test_outputs_and_overlaps():
    q = torch.zeros((4, 6, 64))
    assert att._output(q, q, (4, 6, 64), "out") is q
    wide = torch.zeros((4, 6, 200))
    assert att._output(wide[:, :, 4:68], q, (4, 6, 64), "out") is not None
    for bad in (q.half(), q[:3], torch.zeros((4, 6, 128))[:, :, ::2], torch.zeros((1, 6, 64)).expand(4, 6, 64),
                torch.zeros((6, 4, 64)).transpose(0, 1), torch.zeros((4, 6, 65))[:, :, :64],
                torch.zeros(4 * 6 * 64 + 1)[1:].view(4, 6, 64)):
        with pytest.raises(ValueError):
            att._output(bad, q, (4, 6, 64), "out")
    buf = torch.zeros((5, 6, 64))
    att._no_overlap(q, q, "q")
    att._no_overlap(buf[:2], buf[3:], "q")
    with pytest.raises(ValueError):
        att._no_overlap(buf[1:], buf[:4], "q")
    att._apart(buf[:2], buf[2:], "out")
    with pytest.raises(ValueError):
        att._apart(buf[:2], buf[1:], "out")


def _c_cache(**kw):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, num_pages=2, kv_heads=2, page_size=16, head_dim=64, kind=0)
    d.update(kw)
    return att._CCache(*(d[f] for f, _ in att._CCache._fields_))


@pytest.mark.parametrize("kw", [dict(k=None), dict(v_scale=None), dict(num_pages=0), dict(kv_heads=0),
                                dict(kv_heads=4097), dict(page_size=24), dict(page_size=8), dict(head_dim=96),
                                dict(kind=2), dict(num_pages=1 << 28)])
def test_c_cache(kw):
    lib, c = hb._lib, _c_cache(**kw)
    p = ctypes.addressof(c)
    assert lib.i4_kv_write_dev(p, 4096, 4096, 128, 64, 128, 64, 1, 0, 4096, None) == -2
    assert "kv_write" in hb.last_error()
    assert lib.i4_kv_read_dev(p, 4096, 4096, 1, 0, 4096, None) == -2
    rc = lib.i4_paged_attention_dev(p, 4096, 128, 64, 1, 2, 0, 4096, 1, 1, 4096, None, 1, 0.1, 4096, 128, 64, None, 0,
                                    None)
    assert rc == -2 and "paged_attention" in hb.last_error()


def test_c_arguments():
    lib, c = hb._lib, _c_cache()
    p = ctypes.addressof(c)
    assert lib.i4_kv_write_dev(None, 4096, 4096, 128, 64, 128, 64, 1, 0, 4096, None) == -2
    for T, dt, k, s in ((-1, 0, 4096, 4096), (1, 3, 4096, 4096), (1, 0, None, 4096), (1, 0, 4096, None),
                        (1 << 30, 0, 4096, 4096)):
        assert lib.i4_kv_write_dev(p, k, 4096, 128, 64, 128, 64, T, dt, s, None) == -2
    assert lib.i4_kv_write_dev(p, None, None, 128, 64, 128, 64, 0, 0, None, None) == 0  # nothing to do

    def attn(q=4096, T=2, heads=4, dt=0, table=4096, cols=1, lens=4096, cu=None, B=2, scale=0.1, out=4096, work=None,
             n=0):
        return lib.i4_paged_attention_dev(p, q, 256, 64, T, heads, dt, table, cols, cols, lens, cu, B, scale, out, 256,
                                          64, work, n, None)

    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(table=None), dict(heads=3), dict(heads=0),
               dict(dt=3), dict(dt=-1), dict(T=3), dict(T=-1), dict(B=-1), dict(cols=-1), dict(cols=1 << 28),
               dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e31), dict(T=1 << 26, B=1 << 26)):
        assert attn(**kw) == -2, kw
    assert attn(T=0, B=0) == 0
    assert attn(cols=4096) == -4 and "workspace" in hb.last_error()
    assert lib.i4_paged_attention_workspace(2, 16, 64, 2, 2, 4, 0, 4096, 0) > 0
    assert lib.i4_paged_attention_workspace(2, 16, 64, 2, 2, 3, 0, 4096, 0) == -2

    def gla(q=4096, T=2, Hk=1, Hv=2, Dk=64, Dv=32, dt=0, cu=None, B=2, so=4096, out=4096, n=0):
        return lib.i4_gated_linear_attention_dev(q, 64, 64, 4096, 64, 64, 4096, 64, 32, 4096, 2, None, 0, T, Hk, Hv, Dk,
                                                 Dv, dt, cu, B, 0.1, None, so, out, 64, 32, None, n, None)

    for kw in (dict(q=None), dict(so=None), dict(out=None), dict(T=-1), dict(B=-1), dict(T=3), dict(Hk=0), dict(Hv=3, Hk=2),
               dict(Hv=70000), dict(Dk=32), dict(Dk=256), dict(Dv=24), dict(Dv=0), dict(Dv=2048), dict(dt=3),
               dict(B=1 << 30, T=1 << 30)):
        assert gla(**kw) == -2, kw
    assert gla(B=0, T=0) == 0
    assert gla(T=100, B=1, cu=4096) == -4 and "workspace" in hb.last_error()
    assert lib.i4_gated_linear_attention_workspace(100, 1, 1, 2, 64, 32, 0, 1, 1) > 0
    assert lib.i4_gated_linear_attention_workspace(100, 1, 1, 2, 64, 24, 0, 1, 1) == -2
