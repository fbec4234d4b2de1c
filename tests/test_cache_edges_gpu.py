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
