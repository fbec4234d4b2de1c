"""The paged cache's calls at values and sizes on the edge of what they take."""
import pytest

import cache_ref as R
from test_cache_gpu import _cache, _case, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("eps", [-1.0, 1e-5])
@pytest.mark.parametrize("dim,rot", [(64, 0), (64, 22), (128, 64), (256, 8)])
def test_append_infinities_past_the_rotated_elements(z2, cuda, name, halves, eps, dim, rot):
    """Elements that are not rotated have no partner: an infinity among them stays (or, normalised, becomes a NaN) and
    leaves its neighbours alone."""
    import torch
    c = _case(cuda, name, new=(5,), cached=(9,), heads=4, kv=2, dim=dim, seed=rot)
    for t in (c["q"], c["new_k"]):
        t.view(5, -1, dim)[:, 0, dim - 1] = float("inf")      # the second of two neighbours
        t.view(5, -1, dim)[1, :, dim - 4] = -float("inf")     # the first
    freq = torch.rand(rot // 2, generator=torch.Generator().manual_seed(1))
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want = R.append(host, 5, c["q"].cpu(), c["new_k"].cpu(), c["new_v"].cpu(), None, None, eps, freq, halves)
    out = torch.zeros_like(c["q"])
    cache = _cache(z2, c)
    z2.cache_append(cache, c["q"], c["new_k"], c["new_v"], out, freq=freq.to(cuda) if rot else None, halves=halves, eps=eps)
    for got, y, tol in ((out, want[0], want[1]), (cache.k_pages, want[2], want[3])):
        got = got.cpu().double()
        assert torch.equal(got.isnan(), y.isnan()) and torch.equal(got.isinf(), y.isinf())
        assert torch.equal(got[y.isinf()], y[y.isinf()])
        _near(got[y.isfinite()], y[y.isfinite()], tol[y.isfinite()])


def _tf32(x):
    """f32 values with the last 13 bits cut off: one tf32 part."""
    import torch
    return (x.float().view(torch.int32) & ~0x1fff).view(torch.float32)


@pytest.mark.parametrize("new,dim,cached", [(1, 64, 700), (1, 128, 1500), (1, 256, 300), (3, 64, 100), (3, 128, 2500), (3, 256, 400), (40, 64, 500),
                                            (40, 128, 2500), (40, 256, 300), (200, 128, 90), (70, 104, 600)])
def test_f32_is_f32(z2, cuda, new, dim, cached):
    """The error in the 2-norm for normal inputs.  It is that of the weights, relatively, as every key's is another.  A product
    of three tf32 parts is off by less than 3 * 2^-20 of it (the product of the lower parts, and either lower part's
    own rounding, 2^-10 * 2^-10 each), a score of about 1 by about as much as one of its products, the exponential by 2^-22, sums
    of 64 elements or 32 keys by at most 8 times 2^-23; twice over for the weights' products with the values: 2^-18 holds
    them all.  One rounded part alone would be off by 2^-11 a product: the last lines show that the bound tells them apart."""
    import torch
    heads, kv = 4, 2
    c = _case(cuda, "f32", new=(new, new), cached=(cached, cached // 3), heads=heads, kv=kv, dim=dim, page=16, seed=dim + new)
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, _ = R.attend_whole(host, c["rows"], c["q"].cpu(), c["out"])
    for max_new in (new, 0):
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], max_new=max_new)
        off = float((c["out"].cpu().double() - want).norm() / want.norm())
        assert off < 2.0 ** -18, off
    one = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    one.k, one.v = _tf32(one.k), _tf32(one.v)
    cut, _ = R.attend_whole(one, c["rows"], _tf32(c["q"].cpu().contiguous()), c["out"])
    assert float((cut - want).norm() / want.norm()) > 2.0 ** -14


@pytest.mark.parametrize("name,new,dim,streams", [("bf16", 1, 64, 3), ("bf16", 1, 256, 3), ("bf16", 60, 64, 2), ("bf16", 60, 128, 160), ("bf16", 60, 256, 2),
                                                  ("f32", 1, 128, 3), ("f32", 60, 64, 2), ("f32", 60, 256, 2)])
def test_values_up_to_the_documented_size(z2, cuda, name, new, dim, streams):
    """Values whose sizes' sum, times 256, just lies within f32, and scores that rise so slowly that the running maximum is
    not raised with each."""
    import torch
    c = _case(cuda, name, new=(new,) * streams, cached=(300,) * streams, heads=2, kv=1, dim=dim, page=16, seed=dim)
    keys = 300 + new
    c["v"].copy_(torch.where(c["v"] >= 0, 1.0, -1.0) * float(2.0 ** 120 / 2 ** (keys - 1).bit_length()))   # sums to 2^120 at most
    ramp = torch.linspace(0.0, 0.2, keys).tolist()
    c["q"].fill_(1.0)
    for s in range(min(streams, 4)):
        for j, x in enumerate(ramp):
            p = int(c["table"][s, j // 16])
            c["k"][p, 0, j % 16] = x
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, tol = R.attend_whole(host, c["rows"], c["q"].cpu(), c["out"])
    for max_new in (new, 0):
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], max_new=max_new)
        _near(c["out"], want, tol)
    assert z2.device_error() == 0
