"""The chunk kernels of the paged cache's attention, at the forms that the launch rules give only to larger calls."""
import pytest

import cache_ref as R
from test_cache_gpu import _cache, _case, _near

pytestmark = pytest.mark.gpu


def _odd_where_none_sees(c, dim, window=0):
    """NaN and infinities, keys' and values', in the slots behind each stream's last token, on pages of no stream and left
    of the first new token's window."""
    import torch
    page, odd = c["k"].shape[2], (float("nan"), float("inf"), -float("inf"))
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    used = torch.zeros(c["k"].shape[0], page, dtype=torch.bool)
    for s in range(len(host.kv_len)):
        first = int(host.kv_len[s]) - int(host.q_start[s + 1] - host.q_start[s])
        for j in range(max(0, first - window + 1) if window else 0, int(host.kv_len[s])):
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
    want, tol = R.attend_whole(host, c["rows"], c["q"].cpu(), c["out"], gate=c["gate"].cpu())
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


# 26 streams of up to 150 new tokens, two query heads to each of six key heads: blocks of 256 rows (two tiles that share
# their keys), known, not known and said too small alike
NEW = [150, 128, 140, 1, 0, 77, 129, 150, 2, 64, 127, 131, 150, 90, 0, 3, 145, 128, 33, 150, 149, 65, 148, 17, 150, 130]
CACHED = [0, 128, 300, 5, 40, 131, 0, 260, 127, 1, 90, 16, 333, 0, 0, 129, 250, 256, 31, 12, 200, 64, 7, 385, 140, 0]


@pytest.mark.parametrize("dim,page,window", [(64, 16, 0), (128, 64, 0), (128, 8, 100), (72, 256, 0), (120, 32, 1), (40, 16, 70)])
def test_blocks_of_256_rows(z2, cuda, dim, page, window):
    """Ragged chunks with holes in their tables, in wider rows, with windows and heads that a tile pads; what no row sees holds
    NaN and infinities, and so do some of a chunk's own tokens, which the rows before them do not see."""
    import torch
    heads, kv = 12, 6
    c = _case(cuda, "bf16", new=NEW, cached=CACHED, heads=heads, kv=kv, dim=dim, page=page, pad=8, extra_rows=2, seed=dim + page,
              holes=((1, 0), (2, 1), (7, 1), (20, 0)))
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    # streams 0, 12 and 22: element 5 of token 130 of the chunk is a NaN, element 6 of token 70 an infinity
    mine = (0, 12, 22)
    odd = [(s, host.place(s, CACHED[s] + 130), host.place(s, CACHED[s] + 70)) for s in mine]
    for _, a, b in odd:
        host.v[a[0], :, a[1], 5] = 0
        host.v[b[0], :, b[1], 6] = 0
    want, tol = R.attend_whole(host, c["rows"], c["q"].cpu(), c["out"], None, window, c["gate"].cpu())
    _odd_where_none_sees(c, dim, window)
    nan, inf = torch.zeros(2, c["rows"], dtype=torch.bool)
    for s, a, b in odd:
        c["v"][a[0], :, a[1], 5] = float("nan")
        c["v"][b[0], :, b[1], 6] = float("inf")
        row = int(host.q_start[s])
        last = row + NEW[s]
        nan[row + 130:min(last, row + 130 + window) if window else last] = True
        inf[row + 70:min(last, row + 70 + window) if window else last] = True
    for max_new in (150, 0, 20):
        c["out"].fill_(7.0)
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], window=window, gate=c["gate"], max_new=max_new)
        got, y, t = (x.cpu().double().view(c["rows"], heads, dim) for x in (c["out"], want, tol))
        assert bool(got[nan][..., 5].isnan().all()) and bool((got[inf][..., 6] == float("inf")).all())
        if max_new == 150:
            whole = torch.ones(c["rows"], heads, dim, dtype=torch.bool)
            whole[nan, :, 5] = False
            whole[inf, :, 6] = False
        _near(got[whole], y[whole], t[whole])
        assert bool((c["out"][sum(NEW):] == 7).all())
    assert z2.device_error() == 0


def test_blocks_of_256_rows_longer_than_said(z2, cuda):
    """Chunks of up to five blocks' rows where the caller says one: each block takes several tiles in turn."""
    import torch
    c = _case(cuda, "bf16", new=[20, 600, 5, 300, 256] + [0, 7] * 20, cached=[700, 150, 0, 129, 1] + [0, 60] * 20, heads=8, kv=4, dim=64, page=16,
              seed=4)
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, tol = R.attend_whole(host, c["rows"], c["q"].cpu(), c["out"], None, 0, c["gate"].cpu())
    _odd_where_none_sees(c, 64)
    first = None
    for max_new in (20, 20, 0, 600):
        c["out"].fill_(7.0)
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], gate=c["gate"], max_new=max_new)
        _near(c["out"], want, tol)
        if max_new == 20:
            first = c["out"].clone() if first is None else first
            assert torch.equal(first, c["out"])
    assert z2.device_error() == 0


@pytest.mark.parametrize("name,dim,streams,new,cached", [("bf16", 64, 26, 150, 100), ("bf16", 128, 26, 150, 0), ("bf16", 128, 1, 150, 300), ("bf16", 256, 2, 60, 200),
                                                         ("bf16", 128, 3, 1, 200), ("f32", 64, 2, 1, 90), ("f32", 128, 2, 40, 90)])
def test_closed_gates(z2, cuda, name, dim, streams, new, cached):
    """Gates of zero: zeros, but not in the place of an infinite value that the row sees (zero times it is no number), and
    rows that see nothing are zeros whatever their gate."""
    import torch
    heads, kv = 12, 6
    c = _case(cuda, name, new=(new,) * streams, cached=(cached,) * streams, heads=heads, kv=kv, dim=dim, page=16)
    c["table"][streams - 1] = -1 if streams > 1 else c["table"][0]
    c["gate"].fill_(-200.0)
    c["gate"][:, 3] = float("nan")
    c["v"][int(c["table"][0, 0]), :, 0, 5] = float("inf")   # stream 0's first token: seen by all of its rows
    for max_new in (new, 0):
        c["out"].fill_(7.0)
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], gate=c["gate"], max_new=max_new)
        got = c["out"].view(-1, heads, dim).cpu()
        if streams > 1:
            assert bool((got[(streams - 1) * new:] == 0).all())
            got = got[:(streams - 1) * new]
        assert bool(got[:, 3].isnan().all())
        rest = torch.ones(len(got), heads, dim, dtype=torch.bool)
        rest[:, 3] = False
        rest[:new, :, 5] = False
        assert bool((got[rest] == 0).all())
        assert bool(got[:new, :, 5].isnan().all())
    assert z2.device_error() == 0


def test_two_calls_at_once(z2, cuda):
    """Chunks of heads of 64, 128 and 256 on two streams side by side, clusters of blocks and blocks alone: the bits of each
    call by itself."""
    import torch
    sides = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i, (dim, streams, new) in enumerate([(64, 2, 60), (64, 12, 100), (128, 3, 40), (256, 2, 90), (256, 20, 30), (64, 40, 130)]):
        c = _case(cuda, "bf16", new=(new,) * streams, cached=(700,) * streams, heads=8, kv=4, dim=dim, page=16, seed=i)
        c["cache"], c["outs"] = _cache(z2, c), [torch.empty_like(c["out"]) for _ in range(2)]
        z2.cache_attend(c["cache"], c["q"], c["out"], gate=c["gate"], max_new=new)
        cases.append((c, new))
    torch.cuda.synchronize()
    for turn in range(10):
        for i in range(len(cases)):
            for k, side in enumerate(sides):
                c, new = cases[(i * (2 * k + 1) + 3 * k + turn) % len(cases)]
                z2.cache_attend(c["cache"], c["q"], c["outs"][k], gate=c["gate"], max_new=new, stream=side)
    torch.cuda.synchronize()
    assert z2.device_error() == 0
    for c, _ in cases:
        for out in c["outs"]:
            assert torch.equal(c["out"], out)
