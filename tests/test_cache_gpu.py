"""The paged cache's append and attention against their definitions in 64 bits (cache_ref)."""
import numpy as np
import pytest

import cache_ref as R

pytestmark = pytest.mark.gpu


def _type(name):
    import torch
    return torch.bfloat16 if name == "bf16" else torch.float32


def _case(cuda, name="bf16", new=(1,), cached=(0,), heads=4, kv=2, dim=64, page=16, pad=0, spare=3, seed=0, extra_rows=0,
          holes=(), shared=False):
    """Tensors of a cache and of a call's token rows; `holes`: (stream, page of it) that are no pages; shared: keys
    and values in one buffer, page by page."""
    import torch
    t = _type(name)
    g = torch.Generator().manual_seed(seed)
    S = len(new)
    wide = max(-(-(n + c) // page) for n, c in zip(new, cached)) + 1
    pages = S * wide + spare
    table = torch.randperm(pages, generator=g)[:S * wide].view(S, wide).to(torch.int32)
    for s, p in holes:
        table[s, p] = -1 if p % 2 else pages
    rows = sum(new) + extra_rows

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    both = normal(pages, 2, kv, page, dim).to(t).to(cuda)
    k, v = (both[:, 0], both[:, 1]) if shared else (both[:, 0].contiguous(), both[:, 1].contiguous())
    c = dict(k=k, v=v, table=table.to(cuda), kv_len=torch.tensor([n + m for n, m in zip(new, cached)], dtype=torch.int32).to(cuda),
             q_start=torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).to(cuda), rows=rows)
    c["q"] = normal(rows, heads * dim + pad).to(t).to(cuda)[:, :heads * dim]
    c["new_k"], c["new_v"] = (normal(rows, kv * dim + pad).to(t).to(cuda)[:, :kv * dim] for _ in range(2))
    c["gate"] = normal(rows, heads + pad).to(t).to(cuda)[:, :heads]
    c["out"] = torch.full((rows, heads * dim + pad), 7.0, dtype=t, device=cuda)[:, :heads * dim]
    return c


def _cache(z2, c):
    return z2.PagedCache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])


def _near(got, want, tol):
    bad = ~((got.cpu().double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got.cpu().double()[bad][:4], want[bad][:4], tol[bad][:4])


def _check_attend(z2, c, scale=None, window=0, gate=True, max_new=0, stream=None):
    import torch
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    gates = c["gate"] if gate else None
    want, tol = R.attend(host, c["rows"], c["q"].cpu(), c["out"], scale, window, c["gate"].cpu() if gate else None)
    z2.cache_attend(_cache(z2, c), c["q"], c["out"], scale=scale, window=window, gate=gates, max_new=max_new, stream=stream)
    torch.cuda.synchronize()
    _near(c["out"], want, tol)
    assert z2.device_error() == 0


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("dim,rot,page", [(64, 64, 16), (128, 128, 64), (128, 32, 8), (96, 42, 16), (256, 256, 32), (8, 8, 8),
                                          (64, 0, 16), (72, 2, 4096)])
def test_append(z2, cuda, name, halves, dim, rot, page):
    import torch
    c = _case(cuda, name, new=(3, 0, 1, 20), cached=(0, 5, 77, 11), dim=dim, page=page, pad=8, extra_rows=2, seed=dim + rot)
    freq = torch.tensor([10000.0 ** (-2 * i / max(rot, 1)) for i in range(rot // 2)], dtype=torch.float32)
    w = [1 + 0.1 * torch.randn(dim) for _ in range(2)]
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    for weights, eps in ((w, 1e-5), ([None, None], 1e-5), ([None, None], -1.0)):
        want = R.append(host, c["rows"], c["q"].cpu(), c["new_k"].cpu(), c["new_v"].cpu(), *weights, eps, freq, halves)
        cache = z2.PagedCache(c["k"].clone(), c["v"].clone(), c["table"], c["kv_len"], c["q_start"])
        out = torch.zeros(c["rows"], c["q"].shape[1], dtype=c["q"].dtype, device=cuda)
        z2.cache_append(cache, c["q"], c["new_k"], c["new_v"], out, freq=freq.to(cuda) if rot else None, halves=halves, eps=eps,
                        q_weight=None if weights[0] is None else weights[0].to(cuda),
                        k_weight=None if weights[1] is None else weights[1].to(cuda))
        _near(out, want[0], want[1])
        _near(cache.k_pages, want[2], want[3])
        assert torch.equal(cache.v_pages.cpu(), want[4])


@pytest.mark.parametrize("halves", [False, True])
def test_append_in_place_and_without_queries(z2, cuda, halves):
    import torch
    c = _case(cuda, "bf16", new=(5, 2), cached=(30, 0), dim=96, pad=16)
    freq = torch.rand(24, device=cuda)
    caches = [z2.PagedCache(c["k"].clone(), c["v"].clone(), c["table"], c["kv_len"], c["q_start"]) for _ in range(3)]
    out = torch.zeros(c["rows"], c["q"].shape[1], dtype=c["q"].dtype, device=cuda)
    z2.cache_append(caches[0], c["q"], c["new_k"], c["new_v"], out, freq=freq, halves=halves)
    z2.cache_append(caches[1], c["q"], c["new_k"], c["new_v"], c["q"], freq=freq, halves=halves)
    z2.cache_append(caches[2], None, c["new_k"], c["new_v"], None, freq=freq, halves=halves)
    assert torch.equal(out, c["q"])
    for other in caches[1:]:
        assert torch.equal(caches[0].k_pages, other.k_pages) and torch.equal(caches[0].v_pages, other.v_pages)


def test_append_far_positions(z2, cuda):
    """A position past 2^20: the angle keeps its digits."""
    import torch
    c = _case(cuda, "f32", new=(3,), cached=(0,), heads=2, kv=1, dim=64, page=4096)
    far = (1 << 20) + 12345
    wide = far // 4096 + 1
    table = torch.full((1, wide), -1, dtype=torch.int32)
    table[0, -1] = 1
    c["table"], c["kv_len"] = table.to(cuda), torch.tensor([far], dtype=torch.int32, device=cuda)
    freq = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float32)
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want = R.append(host, 3, c["q"].cpu(), c["new_k"].cpu(), c["new_v"].cpu(), None, None, 1e-5, freq, False)
    out = torch.zeros_like(c["q"])
    cache = _cache(z2, c)
    z2.cache_append(cache, c["q"], c["new_k"], c["new_v"], out, freq=freq.to(cuda))
    _near(out, want[0], want[1])
    _near(cache.k_pages, want[2], want[3])


def test_append_nowhere(z2, cuda):
    """Tokens on no page, past the table or before the stream's start are written nowhere."""
    import torch
    c = _case(cuda, "bf16", new=(4, 6, 3), cached=(14, 0, 0), page=8, holes=((0, 2),))
    c["kv_len"][1] = c["table"].shape[1] * 8 + 3     # the last three past the table
    c["kv_len"][2] = 1                                # two of three at negative positions
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want = R.append(host, c["rows"], None, c["new_k"].cpu(), c["new_v"].cpu(), None, None, -1.0, None, False)
    cache = _cache(z2, c)
    z2.cache_append(cache, None, c["new_k"], c["new_v"], None, eps=-1.0)
    assert torch.equal(cache.k_pages.cpu().double(), want[2]) and torch.equal(cache.v_pages.cpu(), want[4])


SHAPES = [   # heads, kv, dim, page: every kernel, groups that divide no tile, sizes between the kernels'
    (4, 4, 64, 16), (8, 2, 128, 16), (6, 2, 128, 32), (4, 1, 96, 8), (3, 1, 256, 64), (5, 5, 8, 8), (16, 1, 64, 128), (7, 1, 128, 256),
    (2, 2, 200, 4096)]


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
def test_attend_one_token(z2, cuda, name, heads, kv, dim, page):
    for cached in ((0,), (1, 0, 15, 16, 17, 130), (900, 3)):
        c = _case(cuda, name, new=(1,) * len(cached), cached=cached, heads=heads, kv=kv, dim=dim, page=page, seed=heads)
        _check_attend(z2, c, max_new=1)


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 37])
def test_attend_chunks(z2, cuda, name, heads, kv, dim, page, window):
    """Chunks of several lengths, a stream without new tokens, rows behind the last stream."""
    c = _case(cuda, name, new=(5, 0, 33, 1, 70), cached=(260, 9, 0, 500, 61), heads=heads, kv=kv, dim=dim, page=page, pad=8,
              extra_rows=3, seed=dim)
    for max_new in (0, 70, 5):   # not known, known, said too small
        _check_attend(z2, c, window=window, gate=max_new != 5, max_new=max_new)


@pytest.mark.parametrize("name,heads,kv,dim", [("bf16", 8, 2, 128), ("bf16", 4, 4, 64), ("bf16", 4, 2, 24), ("bf16", 6, 3, 104),
                                               ("bf16", 4, 2, 136), ("bf16", 4, 1, 256), ("bf16", 5, 5, 192), ("f32", 4, 2, 128), ("f32", 3, 1, 72)])
def test_attend_long_chunks(z2, cuda, name, heads, kv, dim):
    """Several tiles to a stream, longer than the caller says."""
    c = _case(cuda, name, new=(300, 129), cached=(140, 0), heads=heads, kv=kv, dim=dim, page=32, seed=3)
    for max_new in (300, 40):
        _check_attend(z2, c, max_new=max_new)


@pytest.mark.parametrize("streams,new,cached", [(1, 40, 3000), (3, 17, 1000), (40, 9, 200), (90, 9, 30)])
def test_attend_wide_heads(z2, cuda, streams, new, cached):
    """Heads past 128 elements in chunks: clusters of eight blocks to a tile, of two, one, and more tiles than SMs."""
    c = _case(cuda, "bf16", new=(new,) * streams, cached=(cached,) * streams, heads=8, kv=2, dim=232, page=8, holes=((0, 1),), seed=2)
    for max_new in (0, new):
        _check_attend(z2, c, max_new=max_new)
    _check_attend(z2, c, window=150, gate=False, scale=0.3)


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_attend_pages_that_are_none(z2, cuda, name, new):
    """Holes in the table (a window's left-behind pages, and others), a stream that sees nothing at all."""
    import torch
    c = _case(cuda, name, new=(new, new, new), cached=(200, 64, 0), heads=4, kv=2, dim=64, page=16, holes=((0, 0), (0, 1), (0, 5), (1, 2)), seed=new)
    c["table"][2] = -1
    for window in (0, 50):
        _check_attend(z2, c, window=window)
    out = c["out"][2 * new:]
    assert bool((out == 0).all())
    # fewer tokens than new rows: the first rows lie before the stream and see nothing
    c["kv_len"][0] = max(new - 2, 0)
    _check_attend(z2, c)
    c["kv_len"][0] = -5
    _check_attend(z2, c)
    c["kv_len"][1] = c["table"].shape[1] * 16 + 2   # tokens past the table are nowhere
    _check_attend(z2, c)
    assert torch.isfinite(c["out"].float()).all()


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("new,dim", [(1, 64), (5, 128), (5, 256), (40, 64), (100, 128), (40, 72), (400, 40)])
def test_attend_odd_values_in_masked_places(z2, cuda, name, new, dim):
    """NaN and infinities past the last token, on other streams' pages, at later tokens of the chunk, left of the
    window and in slots that hold none: rows that do not see them are as without them; rows that see a NaN value have it."""
    import torch
    group = 8 if new > 1 else 2
    c = _case(cuda, name, new=(new, new), cached=(150, 33), heads=group, kv=1, dim=dim, page=16, seed=new + dim)
    odd = (float("nan"), float("inf"), -float("inf"))
    window = 64
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, tol = R.attend(host, c["rows"], c["q"].cpu(), c["out"], None, window, c["gate"].cpu())
    used = torch.zeros(c["k"].shape[0], 16, dtype=torch.bool)
    for s in range(2):
        for j in range(int(host.kv_len[s])):
            first = int(host.kv_len[s]) - new
            if j > first - window:   # seen by some row
                p, slot = host.place(s, j)
                used[p, slot] = True
    for i, (p, slot) in enumerate((~used).nonzero().tolist()):
        c["k"][p, 0, slot, i % dim] = odd[i % 3]
        c["v"][p, 0, slot, (3 * i) % dim] = odd[(i + 1) % 3]
        c["v"][p, 0, slot, (3 * i + 1) % dim] = odd[i % 3]
    z2.cache_attend(_cache(z2, c), c["q"], c["out"], window=window, gate=c["gate"])
    _near(c["out"], want, tol)
    if new > 1:   # the last token of stream 0: only its own rows see it
        p, slot = host.place(0, int(host.kv_len[0]) - 1)
        c["v"][p, 0, slot, 5] = float("nan")
        c["v"][p, 0, slot, 6] = float("inf")
        c["k"][p, 0, slot, 1] = float("nan") if new == 5 else c["k"][p, 0, slot, 1]
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], window=window, gate=c["gate"])
        keep = torch.ones(c["rows"], dtype=torch.bool)
        keep[new - 1] = False
        _near(c["out"][keep.to(cuda)], want[keep], tol[keep])
        last = c["out"][new - 1].view(group, dim).float().cpu()
        assert torch.isnan(last[:, 5]).all() and not torch.isfinite(last[:, 6]).any()
        if new != 5:
            rest = torch.ones(dim, dtype=torch.bool)
            rest[5] = rest[6] = False
            assert torch.isfinite(last[:, rest]).all()


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("new,dim", [(1, 64), (3, 128), (5, 256), (40, 64), (40, 128), (90, 256), (400, 128), (70, 40)])
def test_attend_seen_infinities(z2, cuda, name, new, dim):
    """Tokens that every row sees: a key whose score is -inf has no weight, an infinite value makes its element infinite,
    and a row's infinite query makes that row alone a NaN."""
    import torch
    c = _case(cuda, name, new=(new,), cached=(150,), heads=4, kv=2, dim=dim, page=16, seed=new + dim)
    c["q"].view(new, 4, dim)[..., 1] = c["q"].view(new, 4, dim)[..., 1].abs() + 0.25
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    place = host.place
    host.place = lambda s, j: None if j in (30, 101) else place(s, j)
    want, tol = R.attend(host, new, c["q"].cpu(), c["out"], None, 0, c["gate"].cpu())
    for j in (30, 101):
        p, slot = place(0, j)
        c["k"][p, :, slot, 1] = -float("inf")
        c["v"][p, :, slot] = 1e30
    (p, slot), (p1, slot1) = place(0, 20), place(0, 149)
    c["v"][p, :, slot, 3], c["v"][p1, :, slot1, 4] = float("inf"), -float("inf")
    z2.cache_attend(_cache(z2, c), c["q"], c["out"], gate=c["gate"])
    got, rest = c["out"].view(new, 4, dim).cpu(), torch.ones(dim, dtype=torch.bool)
    assert bool((got[..., 3] == float("inf")).all()) and bool((got[..., 4] == -float("inf")).all())
    rest[3] = rest[4] = False
    _near(got[..., rest], want.view(new, 4, dim)[..., rest], tol.view(new, 4, dim)[..., rest])
    c["q"].view(new, 4, dim)[new - 1, 2, 5] = float("inf")
    z2.cache_attend(_cache(z2, c), c["q"], c["out"], gate=c["gate"])
    again = c["out"].view(new, 4, dim).cpu()
    assert bool(again[new - 1, 2].isnan().all())
    keep = torch.ones(new, 4, dtype=torch.bool)
    keep[new - 1, 2] = False
    _near(again[keep][:, rest], want.view(new, 4, dim)[keep][:, rest], tol.view(new, 4, dim)[keep][:, rest])
    assert z2.device_error() == 0


@pytest.mark.parametrize("name,new,heads", [("bf16", 1, 4), ("bf16", 40, 4), ("bf16", 300, 4), ("f32", 1, 4), ("f32", 3, 2), ("f32", 40, 4)])
def test_last_positions(z2, cuda, name, new, heads):
    """The last tokens that a stream can have, 2^31 - 256 of them, all others on no page: as the same tokens on a
    stream's first page."""
    import torch
    page, last = 4096, 2 ** 31 - 256
    c = _case(cuda, name, new=(new,), cached=(page - 256 - new,), heads=heads, kv=2, dim=64, page=page, seed=new)
    c["table"] = c["table"][:, :1]
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, tol = R.attend(host, c["rows"], c["q"].cpu(), c["out"], None, 40, c["gate"].cpu())
    table = torch.full((1, 2 ** 31 // page), -1, dtype=torch.int32)
    table[0, -1] = int(c["table"][0, 0])
    c["table"], c["kv_len"] = table.to(cuda), torch.tensor([last], dtype=torch.int32).to(cuda)
    for max_new in (0, new):
        c["out"].fill_(7.0)
        z2.cache_attend(_cache(z2, c), c["q"], c["out"], window=40, gate=c["gate"], max_new=max_new)
        _near(c["out"], want, tol)
    freq = (10000.0 ** (-torch.arange(32) / 32) / 8).float()
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    want, tol, keys, k_tol, values = R.append(host, new, c["q"].cpu(), c["new_k"].cpu(), c["new_v"].cpu(), None, None, 1e-5,
                                              freq, False)
    z2.cache_append(_cache(z2, c), c["q"], c["new_k"], c["new_v"], c["out"], freq=freq.to(cuda))
    _near(c["out"], want, tol)
    _near(c["k"], keys, k_tol)
    assert torch.equal(c["v"].cpu(), values)
    assert z2.device_error() == 0


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 4, 50])
def test_attend_large_scores(z2, cuda, name, new):
    """Scores of thousands that rise from key to key: the running maximum is raised again and again."""
    c = _case(cuda, name, new=(new,), cached=(700,), heads=4, kv=1, dim=64, page=16, seed=9)
    import torch
    ramp = torch.linspace(0.1, 30.0, 760 // 16 + 2).tolist()
    for i, p in enumerate(c["table"][0].tolist()):
        c["k"][p] = c["k"][p].sign() * ramp[min(i, len(ramp) - 1)]
    c["q"].copy_(c["q"].sign() * 8)
    host = R.Cache(c["k"], c["v"], c["table"], c["kv_len"], c["q_start"])
    # the inputs are powers of two times few-bit numbers in bf16; scores are exact to 2^-16 of their terms all the same
    want, tol = R.attend(host, c["rows"], c["q"].cpu(), c["out"])
    z2.cache_attend(_cache(z2, c), c["q"], c["out"], max_new=new)
    _near(c["out"], want, tol)


def test_attend_keys_and_values_in_one_buffer(z2, cuda):
    for name in ("bf16", "f32"):
        for new in (1, 6, 64):
            c = _case(cuda, name, new=(new,), cached=(90,), heads=4, kv=2, dim=128, page=32, shared=True)
            _check_attend(z2, c)


def test_attend_offsets_past_32_bits(z2, cuda):
    """Pages whose elements lie past 2^31 from the cache's start."""
    import torch
    for name, new, dim in (("bf16", 1, 128), ("bf16", 40, 128), ("f32", 1, 64), ("f32", 40, 64)):
        t, page, pages = _type(name), 4096, (1 << 31) // (4096 * dim) + 3
        k = torch.zeros(pages, 1, page, dim, dtype=t, device=cuda)
        v = torch.zeros(pages, 1, page, dim, dtype=t, device=cuda)
        g = torch.Generator(device="cuda").manual_seed(1)
        k[-1].normal_(generator=g)
        v[-1].normal_(generator=g)
        c = dict(k=k, v=v, table=torch.tensor([[pages - 1]], dtype=torch.int32, device=cuda),
                 kv_len=torch.tensor([100], dtype=torch.int32, device=cuda), q_start=torch.tensor([0, new], dtype=torch.int32, device=cuda),
                 rows=new, q=torch.randn(new, 2 * dim, device=cuda).to(t), gate=torch.randn(new, 2, device=cuda).to(t),
                 out=torch.zeros(new, 2 * dim, dtype=t, device=cuda))
        small = R.Cache(k[-1:], v[-1:], torch.zeros(1, 1, dtype=torch.int32), c["kv_len"], c["q_start"])
        want, tol = R.attend(small, new, c["q"].cpu(), c["out"], gate=c["gate"].cpu())
        cache = _cache(z2, c)
        z2.cache_attend(cache, c["q"], c["out"], gate=c["gate"])
        _near(c["out"], want, tol)
        row = torch.randn(new, dim, device=cuda).to(t)
        z2.cache_append(cache, None, row, row, None, eps=-1.0)
        assert torch.equal(v[-1, 0, 100 - new:100], row)
        del k, v, c, cache
        torch.cuda.empty_cache()


def test_many_streams(z2, cuda):
    """More streams than a block has threads, most of them without new tokens."""
    S = 1500
    r = np.random.default_rng(0)
    new = [int(x) for x in (r.random(S) < 0.2) * r.integers(1, 4, S)]
    c = _case(cuda, "bf16", new=new, cached=[int(x) for x in r.integers(0, 40, S)], heads=2, kv=1, dim=64, page=8)
    for max_new in (3, 0):
        _check_attend(z2, c, max_new=max_new)
    c = _case(cuda, "bf16", new=[40 if i == 700 else n for i, n in enumerate(new)], cached=[0] * S, heads=2, kv=1, dim=64, page=8)
    _check_attend(z2, c, max_new=40)


def test_starts_that_make_no_sense(z2, cuda):
    """Starts that fall, lie outside the rows or a length past everything: nothing outside the buffers is touched."""
    import torch
    for name in ("bf16", "f32"):
        for new in (2, 60):
            c = _case(cuda, name, new=(new, new, new), cached=(20, 40, 0), heads=4, kv=2, dim=64, extra_rows=1)
            guard = torch.full((c["rows"] + 2, 4 * 64), 3.0, dtype=c["q"].dtype, device=cuda)
            for starts in ((5, 0, 10 ** 6, -7), (-3, new, new // 2, 2 ** 31 - 1), (0, 0, 0, 0)):
                c["q_start"].copy_(torch.tensor(starts, dtype=torch.int32))
                c["kv_len"].copy_(torch.tensor([2 ** 31 - 1, -2 ** 31, 30], dtype=torch.int32))
                for max_new in (1, new):
                    z2.cache_attend(_cache(z2, c), c["q"], guard[1:-1], gate=c["gate"], max_new=max_new)
                z2.cache_append(_cache(z2, c), c["q"], c["new_k"], c["new_v"], guard[1:-1])
            torch.cuda.synchronize()
            assert bool((guard[0] == 3).all()) and bool((guard[-1] == 3).all())
            assert z2.device_error() == 0


def test_streams_graphs_and_repeats(z2, cuda):
    """Calls on a stream of their own, captured and replayed on new inputs, equal from run to run."""
    import torch
    for name, new, max_new in (("bf16", 1, 1), ("bf16", 5, 5), ("bf16", 80, 80), ("f32", 1, 1), ("f32", 30, 30)):
        c = _case(cuda, name, new=(new, new), cached=(333, 50), heads=8, kv=2, dim=128, page=16)
        cache = _cache(z2, c)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        q_out = torch.zeros(c["rows"], 8 * 128, dtype=c["q"].dtype, device=cuda)
        freq = torch.rand(64, device=cuda)

        def step(stream=None):
            z2.cache_append(cache, c["q"], c["new_k"], c["new_v"], q_out, freq=freq, stream=stream)
            z2.cache_attend(cache, q_out, c["out"], gate=c["gate"], max_new=max_new, stream=stream)

        step(side)
        side.synchronize()
        first, k1 = c["out"].clone(), c["k"].clone()
        c["out"].zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, c["out"]) and torch.equal(k1, c["k"])
        c["new_k"].normal_()
        c["kv_len"] -= 3
        graph.replay()
        torch.cuda.synchronize()
        again = c["out"].clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(again, c["out"]) and not torch.equal(first, again)
