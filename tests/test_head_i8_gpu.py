"""The 8-bit head against whole-number arithmetic and 64 bits."""
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _rounded(x):
    """(q, scale) of rows x (values that f32 holds) by the definition: 127 x / max |x| to the nearest integer, ties to
    even, in exact fractions."""
    q, scale = np.zeros(x.shape, np.int64), np.zeros(len(x))
    for r, row in enumerate(x):
        if not np.isfinite(row).all():
            scale[r] = np.nan
            continue
        most = Fraction(float(np.abs(row).max()))
        if most == 0:
            continue
        if r < 30 or r % 100 == 0:
            q[r] = [round(127 * Fraction(float(v)) / most) for v in row]
        else:   # (in 64 bits: no random row has a tie that they would not show)
            q[r] = np.rint(127 * row.astype(np.float64) / float(most))
        scale[r] = float(most / 127)
    return q, scale


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim,pad", [(1, 16, 0), (7, 33, 0), (5, 130, 3), (3, 1024, 8), (2, 6001, 0), (2, 8192, 16), (1300, 40, 0),
                                          (1185, 2600, 8)])
def test_quantize_rows(z2, cuda, name, rows, dim, pad):
    import torch
    t = torch.bfloat16 if name == "bf16" else torch.float32
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(rows, dim + pad, generator=g) * 10.0 ** torch.randint(-6, 6, (rows, 1), generator=g)
    x = x.to(t)
    x[:, 1::5] = (torch.randint(-127, 128, x[:, 1::5].shape, generator=g).float() / 2).to(t)   # ties, where the largest is 63.5
    x[0] = x[0].clamp(-63.5, 63.5)
    x[0, 0] = 63.5
    if rows > 2:
        x[1] = 0
        x[2, dim // 2] = float("inf") if rows > 4 else float("nan")
    if rows > 4:
        x[3] = (x[3].float() * 1e-38).to(t)   # subnormals among them
        x[4] = (x[4].float().sign() * 3e38).to(t)
    d = x.to(cuda)[:, :dim]
    q, s = torch.empty(rows, dim, dtype=torch.int8, device=cuda), torch.empty(rows, device=cuda)
    z2.quantize_rows(d, q, s)
    want, scale = _rounded(x[:, :dim].float().numpy())
    assert np.array_equal(q.cpu().numpy().astype(np.int64), want)
    got = s.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(scale))
    ok = ~np.isnan(scale)
    # one f32 rounding; below the normal range half of the smallest step
    assert np.all(np.abs(got - scale)[ok] <= 2.0 ** -24 * scale[ok] + 2.0 ** -150)


def _head(z2, cuda, name, batch, n_cb, vocab, rows, dim, softcap=15.0, seed=0, odd=False, offset=0):
    import torch
    t = torch.bfloat16 if name == "bf16" else torch.float32
    g = torch.Generator().manual_seed(seed + batch)
    W = torch.randint(-127, 128, (n_cb * rows, dim), generator=g, dtype=torch.int8)
    ws = torch.rand(n_cb * rows, generator=g) * 2e-3 + 1e-4
    h = (torch.randn(batch, dim, generator=g) * (0.1 + 3 * torch.rand(batch, 1, generator=g))).to(t)
    if odd and batch > 1:
        h[batch // 2, dim - 1] = float("nan")
    out = torch.full((batch * n_cb * vocab + offset,), 5.0, device=cuda)[offset:].view(batch, n_cb, vocab)
    work = torch.empty(z2.head_i8_work(batch, dim), dtype=torch.uint8, device=cuda)
    z2.head_i8(W.to(cuda), ws.to(cuda), rows, n_cb, vocab, h.to(cuda), out, work, softcap=softcap)
    torch.cuda.synchronize()
    assert z2.device_error() == 0
    x = h.double()
    bad = ~torch.isfinite(x).all(1)
    most = torch.where(bad, 1.0, x.abs().amax(1))
    q = torch.round(127 * torch.where(bad[:, None], 0.0, x) / most[:, None])   # (ties: no random row has one)
    keep = torch.cat([torch.arange(c * rows, c * rows + vocab) for c in range(n_cb)])
    y = (q @ W[keep].double().t()) * (most / 127)[:, None] * ws[keep].double()
    y = softcap * torch.tanh(y / softcap) if softcap > 0 else y
    y = y.view(batch, n_cb, vocab)
    got = out.cpu().double()
    assert torch.isnan(got[bad]).all()
    # the sum's rounding to f32, two products and the scale's own: 2^-22; the softcap 2^-21
    err = (got - y).abs()[~bad]
    assert bool((err <= 2.0 ** -20 * y.abs()[~bad]).all()), float((err / y.abs()[~bad].clamp(min=1e-30)).max())


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("batch", [1, 2, 15, 16, 17, 64, 65, 130, 257, 600])
def test_head_i8(z2, cuda, name, batch):
    _head(z2, cuda, name, batch, 9, 1024, 1026, 256, odd=batch > 60)


@pytest.mark.parametrize("n_cb,vocab,rows,dim", [(1, 1, 1, 16), (1, 63, 63, 48), (3, 65, 70, 2048), (2, 129, 129, 1040), (5, 257, 300, 144),
                                                 (1, 5000, 5000, 128), (16, 33, 35, 4112)])
@pytest.mark.parametrize("batch", [1, 33, 300])
def test_head_i8_sizes(z2, cuda, n_cb, vocab, rows, dim, batch):
    _head(z2, cuda, "bf16", batch, n_cb, vocab, rows, dim, seed=7)
    _head(z2, cuda, "f32", batch, n_cb, vocab, rows, dim, softcap=0.0, seed=8, offset=1)


def test_head_i8_full_batch(z2, cuda):
    _head(z2, cuda, "bf16", 4096, 9, 1024, 1026, 2048, odd=True)


def test_head_i8_largest_sums(z2, cuda):
    """The deepest row, all products 127 * 127: the sum is near the end of 32 bits."""
    import torch
    dim = 131072
    W = torch.full((16, dim), 127, dtype=torch.int8, device=cuda)
    W[1::2] = -127
    h = torch.ones(3, dim, device=cuda)
    h[1] = -2.0
    out = torch.empty(3, 1, 16, device=cuda)
    work = torch.empty(z2.head_i8_work(3, dim), dtype=torch.uint8, device=cuda)
    z2.head_i8(W, torch.ones(16, device=cuda), 16, 1, 16, h, out, work, softcap=0.0)
    want = torch.tensor([1.0, -2.0, 1.0], dtype=torch.float64)[:, None] * torch.tensor([127.0, -127.0] * 8, dtype=torch.float64) * dim
    got = out[:, 0].cpu().double()
    assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs()).all())


def test_head_i8_ends_of_the_softcap(z2, cuda):
    """Products past f32 and near nothing: the softcap's ends, its sign, and zeros for rows of zeros."""
    import torch
    W = torch.full((64, 32), 100, dtype=torch.int8, device=cuda)
    W[1::2] = -100
    h = torch.tensor([[3e38], [1e-3], [0.0], [1e-44]], device=cuda).expand(4, 32).contiguous()
    out = torch.empty(4, 1, 64, device=cuda)
    work = torch.empty(z2.head_i8_work(4, 32), dtype=torch.uint8, device=cuda)
    z2.head_i8(W, torch.full((64,), 100.0, device=cuda), 64, 1, 64, h, out, work)
    out = out[:, 0].cpu()
    assert torch.equal(out[0], torch.tensor([15.0, -15.0] * 32))
    assert torch.equal(out[2], torch.zeros(64)) and bool((out[3].abs() < 1e-30).all())
    assert bool((out[1, ::2] > 0).all()) and torch.equal(out[1, ::2], -out[1, 1::2])


def test_head_i8_captured_and_on_streams(z2, cuda):
    """Two captured heads with scratch of their own on two streams, replayed together."""
    import torch
    g = torch.Generator().manual_seed(0)
    W = torch.randint(-127, 128, (1024, 512), generator=g, dtype=torch.int8).to(cuda)
    ws = torch.rand(1024, generator=g).to(cuda) * 1e-3
    jobs = []
    for batch in (3, 700):
        h = torch.randn(batch, 512, generator=g).to(cuda)
        work = torch.empty(z2.head_i8_work(batch, 512), dtype=torch.uint8, device=cuda)
        out, want = torch.empty(batch, 4, 256, device=cuda), torch.empty(batch, 4, 256, device=cuda)
        z2.head_i8(W, ws, 256, 4, 256, h, want, work)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            z2.head_i8(W, ws, 256, 4, 256, h, out, work)
        jobs.append((graph, out, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, out, _, stream in jobs:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in jobs:
        assert torch.equal(out, want)
