"""The block-tail norm against its formula in 64 bits."""
import numpy as np
import pytest

import operators_ref as R

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
# Relative error of a normed element before its store, in half steps of f32: the sum of squares
# (45 additions at most on any one path: 8 or 4 elements, 5 lanes, 32 warps; the root halves it),
# the root's 2 ulp, exponential, sum and reciprocal of the sigmoid 4 ulp, its argument |g| < 6 ulp
# in bf16, the products 4 half steps: 23 + 4 + 8 + 12 + 4.
REL = 51 * F


def _tensors(cuda, rows, dim, dtype, gate, pad=0, seed=0):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    t = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]

    def cut(scale):
        return (torch.randn(rows, dim + pad, generator=g, device=cuda) * scale).to(t)[:, :dim]

    shape = {"none": None, "full": (rows, dim), "row": (rows, 1), "column": (1, dim),
             "one": (1, 1)}[gate]
    gates = None if shape is None else torch.randn(shape, generator=g, device=cuda).to(t)
    w = [1 + 0.1 * torch.randn(dim, generator=g, device=cuda) for _ in range(2)]
    return cut(2.0), cut(1.0), gates, w


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _check(x, y, gate, sigmoid, w, post_eps, scale, norm_eps, r, n):
    half = 2.0 ** -8 if x.element_size() == 2 else F   # of the store
    want_r, want_n, mag = R.block_norm(_np(x), _np(y), _np(w[0]), post_eps, _np(gate), sigmoid, scale,
                                       _np(w[1]), norm_eps)
    err = REL * mag + F * np.abs(want_r)
    if r is not None:
        assert (np.abs(_np(r) - want_r) <= err + half * np.abs(want_r) + 1e-40).all()
    if n is not None:
        # r's error moves an element and, by the row's, the root
        rms = np.sqrt((want_r * want_r).mean(1, keepdims=True) + norm_eps)
        rel = np.sqrt((err * err).mean(1, keepdims=True)) / rms
        bound = err / rms * (1 if w[1] is None else np.abs(_np(w[1]))) + (rel + REL) * np.abs(want_n)
        assert (np.abs(_np(n) - want_n) <= bound * 1.01 + half * np.abs(want_n) + 1e-40).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim,pad", [(1, 2048, 0), (1, 1, 0), (3, 7, 2), (5, 8, 8), (300, 32, 0),
                                          (4000, 64, 0), (257, 2048, 64), (600, 520, 0), (2, 8192, 0),
                                          (2, 8200, 0), (3, 5003, 1), (1000, 257, 3), (40, 1000, 24)])
def test_shapes(z2, cuda, dtype, rows, dim, pad):
    """Vector and element-wise kernels, several rows to a block, rows past one wave, odd strides."""
    import torch
    x, y, g, w = _tensors(cuda, rows, dim, dtype, "full", pad, rows + dim)
    r, n = (torch.empty(rows, dim, dtype=x.dtype, device=cuda) for _ in range(2))
    z2.block_norm(x, y, r, n, post_weight=w[0], gate=g, gate_sigmoid=True, scale=0.7, norm_weight=w[1])
    _check(x, y, g, True, w, 1e-5, 0.7, 1e-5, r, n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [96, 99])
@pytest.mark.parametrize("gate", ["none", "full", "row", "column", "one"])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_parts(z2, cuda, dtype, dim, gate, sigmoid):
    """Every gate with and without sigmoid, weights, first norm and either output missing."""
    import torch
    x, y, g, w = _tensors(cuda, 17, dim, dtype, gate, 0, dim)
    for post_eps, weights, outs in ((1e-5, w, (1, 1)), (-1.0, [None, w[1]], (0, 1)),
                                    (0.0, [w[0], None], (1, 0)), (-1.0, [None, None], (1, 1))):
        r, n = (torch.empty(17, dim, dtype=x.dtype, device=cuda) if o else None for o in outs)
        z2.block_norm(x, y, r, n, post_weight=weights[0], post_eps=post_eps, gate=g,
                      gate_sigmoid=sigmoid, scale=-0.3, norm_weight=weights[1], norm_eps=1e-6)
        _check(x, y, g, sigmoid, weights, post_eps, -0.3, 1e-6, r, n)


@pytest.mark.parametrize("dim", [256, 255])
def test_in_place_and_untouched(z2, cuda, dim):
    """r over the residual and n over the block's output, in wider rows whose rest stays."""
    import torch
    rows, wide = 700, 272
    base = [torch.randn(rows + 2, wide, device=cuda).bfloat16() for _ in range(2)]
    kept = [b.clone() for b in base]
    x, y = (b[1:-1, :dim] for b in base)
    x0, y0 = x.clone(), y.clone()
    w = [None, torch.rand(dim, device=cuda) + 0.5]
    z2.block_norm(x, y, x, y, norm_weight=w[1])
    _check(x0, y0, None, False, w, 1e-5, 1.0, 1e-5, x, y)
    for b, k in zip(base, kept):
        assert torch.equal(b[:, dim:], k[:, dim:])
        assert torch.equal(b[0], k[0]) and torch.equal(b[-1], k[-1])


@pytest.mark.parametrize("dim", [64, 63])
def test_edges(z2, cuda, dim):
    """A zero row under eps stays zero, an infinite gate value's sigmoid is 0 or 1, a NaN stays in
    its row, and no rows are no work."""
    import torch
    x = torch.zeros(4, dim, device=cuda)
    y = torch.zeros(4, dim, device=cuda)
    y[1] = 3.0
    y[2, 5] = float("nan")
    y[3] = 1.0
    g = torch.full((4, dim), 200.0, device=cuda)
    g[3] = -float("inf")
    r, n = torch.empty_like(x), torch.empty_like(x)
    z2.block_norm(x, y, r, n, gate=g, gate_sigmoid=True)
    assert (r[0] == 0).all() and (n[0] == 0).all()
    # 1e-5 beside the squares' mean of 9 and 1
    assert torch.allclose(r[1], torch.ones_like(r[1]), rtol=1e-6 + REL, atol=0)
    assert torch.allclose(n[1], torch.ones_like(r[1]), rtol=6e-6 + 2 * REL, atol=0)
    assert torch.isnan(r[2]).all() and torch.isnan(n[2]).all()
    assert (r[3] == 0).all() and (n[3] == 0).all()
    z2.block_norm(x[:0], y[:0], r[:0], n[:0])


def test_captured_on_its_own_stream(z2, cuda):
    """Recorded once and replayed on new inputs; and on a stream that is not the current one."""
    import torch
    x, y, g, w = _tensors(cuda, 33, 512, "bf16", "row", 0, 4)
    r, n = (torch.empty(33, 512, dtype=x.dtype, device=cuda) for _ in range(2))

    def call(stream=None):
        z2.block_norm(x, y, r, n, post_weight=w[0], gate=g, gate_sigmoid=True, norm_weight=w[1], stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    side.synchronize()
    _check(x, y, g, True, w, 1e-5, 1.0, 1e-5, r, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in (5, 6):
        for a, b in zip((x, y, g), _tensors(cuda, 33, 512, "bf16", "row", 0, seed)):
            a.copy_(b)
        graph.replay()
        _check(x, y, g, True, w, 1e-5, 1.0, 1e-5, r, n)
