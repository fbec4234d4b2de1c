"""Argument checks of the paged cache's calls and of the 8-bit head: they come before CUDA is touched, so none of this
needs a GPU."""
import ctypes as C

import pytest

P = 1 << 20   # an address that is never read


def _struct(z2, **kw):
    a = dict(k=P, v=2 * P, dtype=z2.BF16, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64, page_stride=2048, table=P,
             n_streams=3, max_pages=4, kv_len=P, q_start=P)
    a.update(kw)
    return z2._Cache(*a.values())


def _append(z2, cache=None, **kw):
    c = _struct(z2, **(cache or {}))
    a = dict(cache=C.addressof(c), rows=5, n_heads=8, q=P, q_stride=512, k=P, k_stride=128, v=P, v_stride=128, q_weight=P, k_weight=P,
             eps=1e-5, freq=P, rot_dim=64, halves=0, q_out=2 * P, q_out_stride=512)
    a.update(kw)
    return z2.lib().zonos2cu_cache_append(*a.values(), None)


def _attend(z2, cache=None, **kw):
    c = _struct(z2, **(cache or {}))
    a = dict(cache=C.addressof(c), rows=5, n_heads=8, q=P, q_stride=512, scale=0.125, window=0, gate=P, gate_stride=8, max_new=0,
             out=2 * P, out_stride=512)
    a.update(kw)
    return z2.lib().zonos2cu_cache_attend(*a.values(), None)


BAD_CACHE = [dict(k=None), dict(v=None), dict(table=None), dict(kv_len=None), dict(q_start=None), dict(dtype=5), dict(n_pages=0),
             dict(page_size=0), dict(n_kv_heads=0), dict(head_dim=0), dict(n_streams=-1), dict(max_pages=0), dict(page_stride=2040),
             dict(table=P + 2), dict(kv_len=P + 1), dict(q_start=P + 2), dict(n_kv_heads=5, page_stride=8192)]
UNSUPPORTED_CACHE = [dict(head_dim=60), dict(head_dim=264, page_stride=1 << 20), dict(page_size=12), dict(page_size=4), dict(page_size=8192, page_stride=1 << 20),
                     dict(page_stride=2052), dict(k=P + 8), dict(v=P + 2), dict(n_kv_heads=5000, page_stride=1 << 30)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_caches(z2, bad):
    assert _append(z2, bad) == z2.EINVAL and _attend(z2, bad) == z2.EINVAL


@pytest.mark.parametrize("bad", UNSUPPORTED_CACHE)
def test_unsupported_caches(z2, bad):
    assert _append(z2, bad, n_heads=5000 if bad.get("n_kv_heads") else 8) == z2.EUNSUPPORTED
    assert _attend(z2, bad, n_heads=5000 if bad.get("n_kv_heads") else 8) == z2.EUNSUPPORTED


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(n_heads=0), dict(n_heads=7), dict(q_stride=504), dict(k=None), dict(k_stride=120), dict(v=None),
    dict(v_stride=100), dict(eps=float("nan")), dict(eps=float("inf")), dict(freq=None), dict(rot_dim=-2), dict(rot_dim=66), dict(rot_dim=31),
    dict(q_out=None), dict(q_out_stride=504), dict(q_out=P, q_out_stride=1024), dict(q_weight=P + 2), dict(k_weight=P + 1), dict(freq=P + 3)])
def test_append_refuses(z2, bad):
    assert _append(z2, **bad) == z2.EINVAL


@pytest.mark.parametrize("bad", [dict(q=P + 8), dict(q_stride=516), dict(k=P + 2), dict(k_stride=132), dict(v=P + 4), dict(v_stride=130),
                                 dict(q_out=P + 8), dict(q_out_stride=514)])
def test_append_unaligned(z2, bad):
    assert _append(z2, **bad) == z2.EUNSUPPORTED


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(n_heads=0), dict(n_heads=9), dict(q=None), dict(q_stride=504), dict(out=None), dict(out_stride=500),
    dict(out=P), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(gate_stride=7), dict(gate=P + 1)])
def test_attend_refuses(z2, bad):
    assert _attend(z2, **bad) == z2.EINVAL


@pytest.mark.parametrize("bad", [dict(q=P + 2), dict(q_stride=516), dict(out=P + 4), dict(out_stride=514), dict(n_heads=65536)])
def test_attend_unsupported(z2, bad):
    assert _attend(z2, **bad) == z2.EUNSUPPORTED


def test_too_many_rows(z2):
    assert _attend(z2, rows=1 << 28) == z2.EUNSUPPORTED and _append(z2, rows=1 << 28) == z2.EUNSUPPORTED
    many = dict(n_streams=1 << 30)
    assert _attend(z2, many) == z2.EUNSUPPORTED and _append(z2, many) == z2.EUNSUPPORTED


def test_no_cache(z2):
    L = z2.lib()
    assert L.zonos2cu_cache_append(None, 5, 8, P, 512, P, 128, P, 128, P, P, 1e-5, P, 64, 0, 2 * P, 512, None) == z2.EINVAL
    assert L.zonos2cu_cache_attend(None, 5, 8, P, 512, 0.125, 0, P, 8, 0, 2 * P, 512, None) == z2.EINVAL


def test_nothing_to_do(z2):
    assert _append(z2, rows=0) == 0 and _attend(z2, rows=0) == 0
    assert _append(z2, dict(n_streams=0)) == 0 and _attend(z2, dict(n_streams=0)) == 0


def _head(z2, **kw):
    a = dict(W=P, w_scale=P, rows_per_cb=1026, n_cb=9, vocab=1024, dim=2048, hidden=P, dtype=z2.BF16, batch=4, softcap=15.0, work=P,
             work_bytes=1 << 20, out=P)
    a.update(kw)
    return z2.lib().zonos2cu_head_i8(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(W=None), dict(w_scale=None), dict(hidden=None), dict(work=None), dict(out=None), dict(dtype=3), dict(rows_per_cb=1000), dict(n_cb=0),
    dict(vocab=0), dict(dim=0), dict(dim=131088), dict(batch=-1), dict(softcap=float("nan")), dict(work_bytes=0), dict(W=P + 8), dict(w_scale=P + 2),
    dict(work=P + 8), dict(hidden=P + 1), dict(hidden=P + 2, dtype=0), dict(out=P + 2)])
def test_head_i8_refuses(z2, bad):
    assert _head(z2, **bad) == z2.EINVAL


def test_head_i8_unsupported_and_work(z2):
    assert _head(z2, dim=2040) == z2.EUNSUPPORTED
    assert _head(z2, n_cb=1 << 20, rows_per_cb=1024) == z2.EUNSUPPORTED
    assert _head(z2, dim=16, batch=1 << 30, work_bytes=1 << 40) == z2.EUNSUPPORTED
    assert _head(z2, batch=0) == 0
    for batch, dim in ((1, 16), (7, 48), (4096, 2048), (2 ** 20, 131072)):
        need = z2.head_i8_work(batch, dim)
        assert batch * (dim + 4) <= need <= batch * (dim + 4) + 80
        assert _head(z2, batch=batch, dim=dim, work_bytes=need - 1) == z2.EINVAL
    for args in ((-1, 16), (1, 0), (1, 131073)):
        with pytest.raises(z2.Zonos2cuError):
            z2.head_i8_work(*args)


def test_quantize_refuses(z2):
    def call(**kw):
        a = dict(x=P, dtype=z2.F32, rows=3, dim=20, stride=20, q=P, scale=P)
        a.update(kw)
        return z2.lib().zonos2cu_quantize_rows(*a.values(), None)
    for bad in (dict(x=None), dict(q=None), dict(scale=None), dict(dtype=4), dict(rows=-1), dict(dim=0), dict(stride=19), dict(x=P + 2),
                dict(scale=P + 1), dict(x=P + 1, dtype=z2.BF16)):
        assert call(**bad) == z2.EINVAL
    assert call(dim=1 << 30, stride=1 << 30) == z2.EUNSUPPORTED
    assert call(rows=0) == 0


def test_python_checks(z2):
    """Shapes, types and devices are looked at before anything is launched."""
    import torch
    bf, i32 = torch.bfloat16, torch.int32
    pages, table = torch.zeros(6, 2, 16, 8, dtype=bf), torch.zeros(3, 2, dtype=i32)
    lens, starts = torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32)

    def cache(**kw):
        a = dict(k=pages, v=pages, table=table, kv_len=lens, q_start=starts)
        a.update(kw)
        return z2.PagedCache(*a.values())
    for kw in (dict(k=pages[0]), dict(v=pages[:5]), dict(v=pages.float()), dict(k=pages.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(v=torch.zeros(6, 3, 16, 8, dtype=bf)[:, :2]), dict(table=table[0]), dict(kv_len=lens[:2]), dict(q_start=starts[:3])):
        with pytest.raises(ValueError):
            cache(**kw)
    for kw in (dict(table=table.long()), dict(kv_len=lens.float()), dict(k=pages.half(), v=pages.half())):
        with pytest.raises(TypeError):
            cache(**kw)

    c, x, kv = cache(), torch.zeros(5, 32, dtype=bf), torch.zeros(5, 16, dtype=bf)
    for args, kw in (((x, kv[:4], kv, x), {}), ((x, kv, kv[:, :8], x), {}), ((x[:, :20], kv, kv, x), {}), ((x, kv, kv, x[:4]), {}),
                     ((None, kv, kv, x), {}), ((x, kv, kv, None), {}), ((x, kv, kv, x), dict(k_weight=torch.zeros(7))),
                     ((x, kv, kv, torch.zeros(32, 5, dtype=bf).t()), {})):
        with pytest.raises(ValueError):
            z2.cache_append(c, *args, **kw)
    for args, kw in (((x.float(), kv, kv, x), {}), ((x, kv, kv.half(), x), {}), ((x, kv, kv, x), dict(freq=torch.zeros(4).double())),
                     ((x, kv, kv, x), {})):   # the last one: host tensors
        with pytest.raises(TypeError):
            z2.cache_append(c, *args, **kw)
    for args, kw in (((x, x[:4]), {}), ((x[:, :30], x[:, :30]), {}), ((x, x.clone()), dict(gate=torch.zeros(5, 3, dtype=bf)))):
        with pytest.raises(ValueError):
            z2.cache_attend(c, *args, **kw)
    for args, kw in (((x, x.float()), {}), ((x, x.clone()), dict(gate=torch.zeros(5, 4))), ((x, x.clone()), {})):
        with pytest.raises(TypeError):
            z2.cache_attend(c, *args, **kw)

    W, ws, h, out = torch.zeros(16, 32, dtype=torch.int8), torch.zeros(16), torch.zeros(4, 32, dtype=bf), torch.zeros(4, 2, 8)
    work = torch.zeros(1024, dtype=torch.uint8)
    for args in ((W[:15], ws, h, out), (W, ws[:15], h, out), (W, ws, h[:, :16], out), (W, ws, h, out[:3])):
        with pytest.raises(ValueError):
            z2.head_i8(args[0], args[1], 8, 2, 8, args[2], args[3], work)
    for args in ((W.float(), ws, h, out), (W, ws.half(), h, out), (W, ws, h.half(), out), (W, ws, h, out.half()), (W, ws, h, out)):
        with pytest.raises(TypeError):
            z2.head_i8(args[0], args[1], 8, 2, 8, args[2], args[3], work)
    with pytest.raises(ValueError):
        z2.quantize_rows(h, W, ws[:4])
    with pytest.raises(TypeError):
        z2.quantize_rows(h, torch.zeros(4, 32), ws[:4])
