"""The chunk kernels of the paged cache's attention, at the forms that the launch rules give only to larger calls."""
import pytest

import cache_ref as R
from test_cache_gpu import _cache, _case, _near

pytestmark = pytest.mark.gpu


def _odd_where_none_sees(c, dim):
    """NaN and infinities, keys' and values', in the slots behind each stream's last token and on pages of no stream."""
    import torch
    page, odd = c["k"].shape[2], (float("nan"), float("inf"), -float("inf"))
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    used = torch.zeros(c["k"].shape[0], page, dtype=torch.bool)
    for s in range(len(host.kv_len)):
        for j in range(int(host.kv_len[s])):
            where = host.place(s, j)
            if where is not None:
                used[where] = True
    for i, (p, slot) in enumerate((~used).nonzero().tolist()):
        c["k"][p, :, slot, i % dim] = odd[i % 3]
        c["v"][p, :, slot, (3 * i) % dim] = odd[(i + 1) % 3]
        c["v"][p, :, slot, (3 * i + 1) % dim] = odd[i % 3]


@pytest.mark.parametrize("dim,streams,cached", [(256, 40, 1000), (256, 25, 700), (256, 1, 6000), (200, 80, 140), (136, 13, 2100)])
def test_wide_heads_over_many_steps(z2, cuda, dim, streams, cached):
    """Heads past 128, steps that every row sees wholly ahead of the last ones, whose masked slots hold NaN and infinities:
    one block to a tile and clusters of two, four and eight, odd and even numbers of steps, the pages spread over more than
    the L2 cache holds where there are many.  The same bits from call to call."""
    import torch
    new = [9 + s % 3 for s in range(streams)]
    c = _case(cuda, "bf16", new=new, cached=[cached + 61 * (s % 7) for s in range(streams)], heads=8, kv=2, dim=dim, page=16,
              spare=3000 if streams > 30 else 3, seed=dim + streams)
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    # the last token of stream 0 is left to its own rows: its value is a NaN
    p, slot = host.place(0, int(host.kv_len[0]) - 1)
    host.v[p, :, slot] = 0
    want, tol = R.attend(host, c["rows"], c["q"].cpu(), c["out"], gate=c["gate"].cpu())
    _odd_where_none_sees(c, dim)
    c["v"][p, :, slot, 7] = float("nan")
    keep = torch.ones(c["rows"], dtype=torch.bool)
    keep[new[0] - 1] = False
    first = None
    for turn in range(40):
        c["out"].fill_(7.0)
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], gate=c["gate"], max_new=max(new))
        if first is None:
            first = c["out"].clone()
            _near(first[keep.to(cuda)], want[keep], tol[keep])
            assert bool(first[new[0] - 1].view(8, dim)[:, 7].isnan().all())
        else:
            assert torch.equal(first.view(torch.int16), c["out"].view(torch.int16)), turn
    assert z2.device_error() == 0
