"""Argument checks of the adapters, the block-tail norm and the draft verification: they come
before CUDA is touched, so none of this needs a GPU."""
import ctypes as C

import numpy as np
import pytest

P = 1 << 20   # an address that is never read


def _params(z2, **kw):
    return z2.SampleParams(**kw)


def _head(z2, **kw):
    a = dict(W=P, dtype=z2.BF16, rows_per_cb=1026, n_cb=9, vocab=1024, dim=2048, hidden=P, batch=4,
             softcap=15.0, A=P, B=P, scale=P, n_adapters=3, rank=16, adapter=P, work=P,
             work_bytes=1 << 30, out=P)
    a.update(kw)
    return z2.lib().zonos2cu_head_adapters(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(W=None), dict(hidden=None), dict(A=None), dict(B=None), dict(adapter=None),
    dict(work=None), dict(out=None), dict(dtype=7), dict(rows_per_cb=1000), dict(n_cb=0),
    dict(vocab=0), dict(dim=0), dict(batch=-1), dict(n_adapters=0), dict(rank=0), dict(rank=257),
    dict(work_bytes=0), dict(softcap=float("nan")), dict(W=P + 1), dict(hidden=P + 1),
    dict(A=P + 1), dict(B=P + 1), dict(scale=P + 2), dict(adapter=P + 2), dict(work=P + 8),
    dict(out=P + 2), dict(dtype=0, W=P + 2)])
def test_head_adapters_refuses(z2, bad):
    assert _head(z2, **bad) == z2.EINVAL


def test_head_adapters_work(z2):
    for dtype in (z2.F32, z2.BF16):
        for batch in (1, 2, 7, 64, 333, 4096):
            for rank in (1, 7, 8, 16, 256):
                need = z2.head_adapters_work(dtype, batch, rank)
                assert 4 * batch * rank <= need <= 8 * batch * rank
                if batch > 1:
                    assert _head(z2, dtype=dtype, batch=batch, rank=rank,
                                 work_bytes=need - 1) == z2.EINVAL
    assert z2.head_adapters_work(z2.BF16, 0, 16) >= 0
    for args in ((9, 4, 16), (z2.BF16, -1, 16), (z2.BF16, 4, 0), (z2.BF16, 4, 257)):
        with pytest.raises(z2.Zonos2cuError):
            z2.head_adapters_work(*args)
    assert _head(z2, batch=0) == 0


def _norm(z2, **kw):
    a = dict(resid=P, block=2 * P, dtype=z2.BF16, rows=4, dim=100, resid_stride=100, block_stride=100,
             post_weight=P, post_eps=1e-5, gate=P, gate_row=100, gate_col=1, sigmoid=1, scale=1.0,
             norm_weight=P, norm_eps=1e-5, resid_out=P, normed_out=2 * P, out_stride=100)
    a.update(kw)
    return z2.lib().zonos2cu_block_norm(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(resid=None), dict(block=None), dict(resid_out=None, normed_out=None), dict(dtype=5),
    dict(rows=-1), dict(dim=0), dict(resid_stride=99), dict(block_stride=99), dict(out_stride=99),
    dict(post_eps=float("nan")), dict(scale=float("inf")), dict(norm_eps=-1.0),
    dict(norm_eps=float("nan")), dict(gate_col=2), dict(gate_row=-100), dict(gate_row=50),
    dict(resid=P + 1), dict(block=P + 1), dict(gate=P + 1), dict(resid_out=P + 1),
    dict(normed_out=P + 1), dict(post_weight=P + 2), dict(norm_weight=P + 2), dict(normed_out=P),
    dict(resid_stride=108), dict(block_stride=108), dict(out_stride=108)])
def test_block_norm_refuses(z2, bad):
    assert _norm(z2, **bad) == z2.EINVAL


def test_block_norm_no_rows(z2):
    assert _norm(z2, rows=0) == 0


def _verify(z2, knobs=None, **kw):
    p = knobs or _params(z2)
    a = dict(logits=P, n_streams=2, n_draft=3, n_cb=9, vocab=1024, stride=1026, params=C.byref(p),
             drafts=P, probs=P, n_drafts=P, uniforms=P, hist=P, hist_len=16, hist_pos=P, allow=P,
             delay=-1, codes=P, n_accepted=P, flags=P)
    a.update(kw)
    return z2.lib().zonos2cu_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(drafts=None), dict(uniforms=None), dict(hist=None), dict(hist_pos=None),
    dict(codes=None), dict(n_accepted=None), dict(params=None), dict(n_streams=-1),
    dict(n_draft=-1), dict(n_draft=4096), dict(n_cb=0), dict(n_cb=17), dict(vocab=0),
    dict(stride=1023), dict(hist_len=-1), dict(logits=P + 2), dict(drafts=P + 2),
    dict(probs=P + 1), dict(n_drafts=P + 2), dict(uniforms=P + 2), dict(hist=P + 2),
    dict(hist_pos=P + 1), dict(allow=P + 2), dict(codes=P + 2), dict(n_accepted=P + 1),
    dict(flags=P + 2)])
def test_verify_drafts_refuses(z2, bad):
    assert _verify(z2, **bad) == z2.EINVAL


def test_verify_drafts_refuses_knobs(z2):
    assert _verify(z2, vocab=1025) == z2.EUNSUPPORTED
    for kw in (dict(temperature=0.0), dict(temperature=float("nan")), dict(top_p=float("nan")),
               dict(min_p=1.5), dict(repetition_penalty=0.0), dict(pad_id=1024)):
        assert _verify(z2, _params(z2, **kw)) == z2.EINVAL
    assert _verify(z2, n_streams=0) == 0


def test_python_checks(z2):
    """The Python entry points look at shapes and types before anything is launched."""
    import torch
    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    x = torch.zeros(4, 32, dtype=bf)
    w = torch.zeros(32)
    for args, kw in (((x, x[:3], x, x), {}), ((x, x, x.float(), x), {}), ((x, x, None, None), {}),
                     ((x, x, x, torch.zeros(4, 64, dtype=bf)[:, :32]), {}),
                     ((x, x, x, x), dict(gate=torch.zeros(4, 31, dtype=bf))),
                     ((x, x, x, x), dict(gate=torch.zeros(4, 32))),
                     ((x, x, x, x), dict(norm_weight=torch.zeros(31))),
                     ((x, x, torch.zeros(32, 4, dtype=bf).t(), None), {})):
        with pytest.raises(ValueError):
            z2.block_norm(*args, **kw)
    with pytest.raises(TypeError):   # no silent path for host tensors
        z2.block_norm(x, x, x, x, norm_weight=w)
    with pytest.raises(TypeError):
        z2.block_norm(x.half(), x.half(), x.half(), None)

    W, A, B = torch.zeros(2 * 8, 32, dtype=bf), torch.zeros(3, 8, 32, dtype=bf), torch.zeros(3, 16, 8, dtype=bf)
    ids, out, work = torch.zeros(4, dtype=i32), torch.zeros(4, 2, 8), torch.zeros(4096, dtype=torch.uint8)

    def head(**kw):
        a = dict(W=W, hidden=x, A=A, B=B, adapter=ids, out=out, scale=None)
        a.update(kw)
        z2.head_adapters(a["W"], z2.BF16, 8, 2, 8, a["hidden"], a["A"], a["B"], a["adapter"], a["out"],
                         work, scale=a["scale"])
    for kw in (dict(W=W[:15]), dict(hidden=x[:, :16]), dict(B=B[:2]), dict(adapter=ids[:3]),
               dict(out=out[:2]), dict(scale=torch.zeros(2)), dict(A=A.transpose(1, 2).contiguous())):
        with pytest.raises(ValueError):
            head(**kw)
    for kw in (dict(adapter=ids.long()), dict(hidden=x.float()), dict(out=out.to(i32)), dict()):
        with pytest.raises(TypeError):
            head(**kw)

    lg, dr, u = torch.zeros(2, 3, 2, 8), torch.zeros(2, 2, 2, dtype=i32), torch.zeros(2, 3, 2, 2)
    codes, n = torch.zeros(2, 3, 2, dtype=i32), torch.zeros(2, dtype=i32)
    p = _params(z2, pad_id=7)
    for bad in ((lg, p, dr[:1], u, codes, n), (lg, p, dr, u[:1], codes, n),
                (lg, p, dr, u, codes[:, :2], n), (lg, p, dr, u, codes, n[:1])):
        with pytest.raises(ValueError):
            z2.verify_drafts(*bad)
    for bad in ((lg, p, dr.long(), u, codes, n), (lg, p, dr, u.double(), codes, n),
                (lg.half(), p, dr, u, codes, n), (lg, p, dr, u, codes, n)):
        with pytest.raises(TypeError):
            z2.verify_drafts(*bad)


def test_context_calls_refuse(z2):
    L = z2.lib()
    buf = np.zeros(16, np.float32).ctypes.data
    assert L.zonos2cu_set_adapters(None, buf, buf, None, 1, 1, z2.F32, 8) == z2.EINVAL
    assert L.zonos2cu_set_stream_adapters(None, None) == z2.EINVAL
