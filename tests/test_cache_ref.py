"""The oracle of the cache's attention by whole products agrees with the one that goes row by row."""
import pytest

import cache_ref as R


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 1, 9])
def test_whole_products(name, window):
    import torch
    from test_cache_gpu import _case
    c = _case("cpu", name, new=(5, 0, 33, 1), cached=(26, 9, 0, 50), heads=6, kv=2, dim=24, page=8, pad=8, extra_rows=3, seed=1,
              holes=((0, 0), (0, 2), (3, 4)))
    c["table"][2, 1] = -1
    c["kv_len"][3] = 0
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    for gate in (None, c["gate"]):
        y, tol = R.attend(host, c["rows"], c["q"], c["out"], 0.3, window, gate)
        z, other = R.attend_whole(host, c["rows"], c["q"], c["out"], 0.3, window, gate)
        assert torch.allclose(y, z, rtol=1e-12, atol=1e-14) and torch.allclose(tol, other, rtol=1e-9, atol=1e-14)
