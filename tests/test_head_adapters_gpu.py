"""The head beside low-rank adapters against its formula in 64 bits, by itself, in a decode
context, and followed by the draft verification."""
import numpy as np
import pytest

import operators_ref as R

pytestmark = pytest.mark.gpu

F = 2.0 ** -24


def _bits(t):
    import torch
    return t.view(torch.int16).cpu().numpy().view(np.uint16)


def _case(cuda, dtype, batch, n_cb, vocab, rows, dim, n, rank, seed=0, low=0.05):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    t = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device=cuda) * by).to(t)

    return dict(W=normal(n_cb * rows, dim, by=0.02), h=normal(batch, dim, by=1.0),
                A=normal(n, rank, dim, by=dim ** -0.5), B=normal(n, n_cb * rows, rank, by=low),
                ids=torch.randint(-1, n + 1, (batch,), generator=g, device=cuda, dtype=torch.int32),
                scale=torch.rand(n, generator=g, device=cuda) + 0.5,
                rows=rows, n_cb=n_cb, vocab=vocab, dtype=dtype)


def _call(z2, c, out=None, work=None, softcap=15.0, scale="own", stream=None):
    import torch
    code = z2.BF16 if c["dtype"] == "bf16" else z2.F32
    batch, rank = len(c["h"]), c["A"].shape[1]
    if out is None:
        out = torch.full((batch, c["n_cb"], c["vocab"]), 7.0, device=c["h"].device)
    if work is None:
        work = torch.full((z2.head_adapters_work(code, batch, rank),), 255, dtype=torch.uint8, device=c["h"].device)
    z2.head_adapters(c["W"], code, c["rows"], c["n_cb"], c["vocab"], c["h"], c["A"], c["B"], c["ids"], out, work,
                     scale=c["scale"] if scale == "own" else None, softcap=softcap, stream=stream)
    return out


def _bound(c, ref, mag, low):
    """The terms' own sizes times a step per addition (2^-23: the tensor cores cut off) beside
    bf16, where A h is kept to f32 by three bf16 parts (2^-24); 4 roundings of each product of
    four and f64 sums beside f32.  The softcap, of slope 1 at most, adds its 1e-5."""
    dim, rank = c["h"].shape[1], c["A"].shape[1]
    steps = 2 * (dim + rank + 8) if c["dtype"] == "bf16" else 8
    return steps * F * (mag + 2 * low) + 1e-5 * np.maximum(1.0, np.abs(ref))


def _check(c, out, softcap=15.0, scale="own", rows=None):
    pick = np.arange(len(c["h"])) if rows is None else np.array(rows)
    np_ = lambda t: t.double().cpu().numpy()
    ids = c["ids"].cpu().numpy()[pick]
    ref, mag, low = R.head_adapters(np_(c["W"]), c["rows"], c["n_cb"], c["vocab"], np_(c["h"])[pick], np_(c["A"]),
                                    np_(c["B"]), ids, np_(c["scale"]) if scale == "own" else None, softcap)
    got = out.double().cpu().numpy()[pick]
    assert (np.abs(got - ref) <= _bound(c, ref, mag, low)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,n_cb,vocab,rows,dim,n,rank", [
    (1, 1, 1, 1, 8, 1, 8), (1, 9, 1024, 1026, 2048, 3, 16), (2, 2, 33, 40, 24, 2, 8), (3, 2, 65, 65, 31, 2, 3),
    (5, 9, 129, 130, 256, 40, 256), (8, 3, 1024, 1024, 72, 1, 1), (64, 2, 200, 200, 512, 64, 40),
    (65, 2, 127, 128, 264, 5, 8), (33, 1, 128, 128, 1000, 4, 24), (130, 3, 70, 72, 64, 200, 12),
    (257, 2, 1001, 1001, 128, 3, 32), (700, 1, 130, 130, 96, 2, 64)])
def test_shapes(z2, cuda, dtype, batch, n_cb, vocab, rows, dim, n, rank):
    """One row to several tiles of them, ranks in and out of eights, sizes that fill no tile, and
    ids on both sides of the range."""
    c = _case(cuda, dtype, batch, n_cb, vocab, rows, dim, n, rank, batch + dim)
    _check(c, _call(z2, c))
    _check(c, _call(z2, c, softcap=0.0, scale=None), 0.0, None)
    assert z2.device_error() == 0


@pytest.mark.parametrize("batch", [3, 40, 200, 600])
@pytest.mark.parametrize("ids", ["none", "same", "one", "alternate", "far"])
def test_ids(z2, cuda, batch, ids):
    """Nobody's, everybody's, one row's and interleaved adapters; ids far outside the range."""
    import torch
    c = _case(cuda, "bf16", batch, 2, 140, 140, 192, 6, 16, batch)
    i = torch.arange(batch, device=cuda, dtype=torch.int32)
    c["ids"] = {"none": i * 0 - 1, "same": i * 0 + 5, "one": torch.where(i == batch // 2, 0, -1).int(),
                "alternate": i % 6, "far": torch.where(i % 2 == 0, 2 ** 31 - 1, -2 ** 31).int()}[ids]
    _check(c, _call(z2, c))


def test_unaligned(z2, cuda):
    """Operands that start inside a 16-byte line."""
    import torch
    for dtype in ("bf16", "f32"):
        c = _case(cuda, dtype, 6, 2, 50, 50, 64, 3, 8, 9)
        for k in ("W", "h", "A", "B"):
            one = dict(c)
            flat = torch.empty(c[k].numel() + 1, dtype=c[k].dtype, device=cuda)
            one[k] = flat[1:].view(c[k].shape)
            one[k].copy_(c[k])
            _check(one, _call(z2, one))


def test_row_without_an_adapter_is_the_heads(z2, cuda):
    """No row gains from the rows beside it: NaN in one adapter reaches only the rows that have it,
    infinite A h reaches its row alone."""
    import torch
    for batch in (5, 100, 520):
        c = _case(cuda, "bf16", batch, 2, 130, 130, 128, 4, 16, batch)
        clean = _call(z2, c)
        c["A"][2, 3, 5] = float("nan")
        got = _call(z2, c)
        hit = c["ids"] == 2
        assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])
        c["A"][2, 3, 5] = 0.0
        c["h"][batch // 2] = 3e38
        got = _call(z2, c)
        rest = torch.arange(batch, device=cuda) != batch // 2
        same = _call(z2, c)
        assert not torch.isnan(got[rest]).any() and torch.equal(got[rest], same[rest])


def test_tensors_elsewhere_are_refused(z2, cuda):
    """A host tensor among device ones is found before anything is launched."""
    import torch
    c = _case(cuda, "bf16", 4, 2, 64, 64, 64, 2, 8, 1)
    for k in ("W", "A", "B", "ids", "scale"):
        with pytest.raises(ValueError):
            _call(z2, dict(c, **{k: c[k].cpu()}))
    with pytest.raises(ValueError):
        _call(z2, c, work=torch.empty(4096, dtype=torch.uint8))
    with pytest.raises(ValueError):
        _call(z2, c, out=torch.empty(4, 2, 64))
    x, w = c["h"], torch.ones(64, device=cuda)
    for args, kw in (((x, x.cpu(), x.clone(), None), {}), ((x, x, x.cpu(), None), {}),
                     ((x, x, x.clone(), None), dict(gate=x.cpu())),
                     ((x, x, x.clone(), None), dict(norm_weight=w.cpu()))):
        with pytest.raises(ValueError):
            z2.block_norm(*args, **kw)
    lg, i32 = torch.zeros(1, 2, 1, 8, device=cuda), torch.int32
    a = [lg, z2.SampleParams(pad_id=7), torch.zeros(1, 1, 1, dtype=i32, device=cuda),
         torch.zeros(1, 2, 1, 2, device=cuda), torch.zeros(1, 2, 1, dtype=i32, device=cuda),
         torch.zeros(1, dtype=i32, device=cuda)]
    for i in (2, 3, 4, 5):
        with pytest.raises(ValueError):
            z2.verify_drafts(*[t.cpu() if j == i else t for j, t in enumerate(a)])


@pytest.mark.parametrize("dtype,batch", [("bf16", 7), ("bf16", 300), ("f32", 5)])
def test_workspace_and_neighbours(z2, cuda, dtype, batch):
    """Exactly the stated scratch, neither side of it nor of the logits written; the same bits
    whatever the scratch held."""
    import torch
    c = _case(cuda, dtype, batch, 2, 100, 104, 128, 3, 16, 3)
    need = z2.head_adapters_work(z2.BF16 if dtype == "bf16" else z2.F32, batch, 16)
    outs = []
    for fill in (0, 255, 127):
        w = torch.full((need + 64,), fill, dtype=torch.uint8, device=cuda)
        flat = torch.full((batch * 200 + 32,), 5.0, device=cuda)
        out = flat[16:-16].view(batch, 2, 100)
        _call(z2, c, out, w[32:32 + need])
        assert (w[:32] == fill).all() and (w[32 + need:] == fill).all()
        assert (flat[:16] == 5.0).all() and (flat[-16:] == 5.0).all()
        outs.append(out.clone())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    z2.head_adapters(c["W"], z2.BF16 if dtype == "bf16" else z2.F32, 104, 2, 100, c["h"][:0], c["A"], c["B"],
                     c["ids"][:0], flat[:0].view(0, 2, 100), torch.empty(0, dtype=torch.uint8, device=cuda))


@pytest.mark.parametrize("dtype,batch", [("bf16", 4), ("bf16", 90), ("bf16", 400), ("f32", 3)])
def test_two_calls_at_once(z2, cuda, dtype, batch):
    """Two captured calls with scratch of their own, replayed on two streams at a time, on new ids."""
    import torch
    cs = [_case(cuda, dtype, batch, 2, 150, 150, 256, 5, 24, i) for i in range(2)]
    code = z2.BF16 if dtype == "bf16" else z2.F32
    outs = [torch.empty(batch, 2, 150, device=cuda) for _ in cs]
    works = [torch.empty(z2.head_adapters_work(code, batch, 24), dtype=torch.uint8, device=cuda) for _ in cs]
    graphs, streams = [torch.cuda.CUDAGraph() for _ in cs], [torch.cuda.Stream() for _ in cs]
    for g, c, o, w in zip(graphs, cs, outs, works):
        with torch.cuda.graph(g):
            _call(z2, c, o, w)
    for turn in range(3):
        for c in cs:
            c["ids"].copy_((c["ids"] + 1 + turn) % 5)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, o in zip(cs, outs):
            _check(c, o)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 6, 150])
@pytest.mark.parametrize("cfg", [None, 1.5])
def test_context_step(z2, oracle, cuda, dtype, S, cfg):
    """zonos2cu_ctx_step with adapters: its logits against the formula (guided ones blended), its
    codes those of the sampler on those logits; then without adapters again."""
    import torch
    from oracle import make_params
    if dtype == "f32" and S > 6:
        S = 20
    n, rank, D = 4, 16, 2048
    c = _case(cuda, dtype, S * (2 if cfg else 1), 9, 1024, 1026, D, n, rank, S, low=0.3)
    code, host = (z2.BF16, _bits) if dtype == "bf16" else (z2.F32, lambda t: t.cpu().numpy())
    ids = np.random.default_rng(S).integers(-1, n, S).astype(np.int32)
    ids[0] = 1
    ctx = z2.Context(0, S, 9, 1024, D, 0, seed=42)
    ctx.set_head(host(c["W"]), code, 1026)
    if cfg:
        ctx.set_cfg(cfg)
    with pytest.raises(z2.Zonos2cuError):
        ctx.set_stream_adapters(ids)
    ctx.set_adapters(host(c["A"]), host(c["B"]), 1026, code, c["scale"].cpu().numpy())
    with pytest.raises(z2.Zonos2cuError):
        ctx.set_stream_adapters(np.full(S, n, np.int32))
    codes = torch.zeros((S, 9), dtype=torch.int32, device=cuda)
    logits = torch.zeros((S, 9, 1024), device=cuda)
    p = z2.SampleParams(0.7, 50, 0.9, 0.02, 1.0, 1023)
    prm = make_params(0.7, 50, 0.9, 0.02, 1.0, 1023)
    np_ = lambda t: t.double().cpu().numpy()
    rng = oracle.rng_seed_streams(42, S)
    for used in (np.full(S, -1, np.int32), ids, None):
        if used is None:
            ctx.set_adapters(None, None, 0, code)
            used = np.full(S, -1, np.int32)
        elif (used >= 0).any():
            ctx.set_stream_adapters(used)
        ctx.step(c["h"], code, p, codes, logits_out=logits)
        torch.cuda.synchronize()
        rows = np.repeat(used, 2) if cfg else used
        ref, mag, low = R.head_adapters(np_(c["W"]), 1026, 9, 1024, np_(c["h"]), np_(c["A"]), np_(c["B"]), rows,
                                        np_(c["scale"]), 15.0)
        bound = _bound(c, ref, mag, low)
        if cfg:
            ref = ref[1::2] + cfg * (ref[0::2] - ref[1::2])
            bound = bound[0::2] * cfg + bound[1::2] * (cfg - 1) + 4 * F * np.abs(ref)
        got = logits.cpu().numpy()
        assert (np.abs(got - ref) <= bound).all()
        oc, _, _ = oracle.step(got, prm, rng, exp_mode=1)   # advances rng
        assert (codes.cpu().numpy() == oc).all()
    assert z2.device_error() == 0
    ctx.close()


@pytest.mark.parametrize("dtype,S,weight", [("f32", 3, True), ("bf16", 5, True), ("bf16", 5, False),
                                            ("bf16", 300, True)])
def test_context_step_with_output_norm(z2, cuda, dtype, S, weight):
    """The norm ahead of head and adapters.  A bf16 head rounds its rows or, folded, the weight's
    products with W and A: 2^-8 of each factor at most."""
    import torch
    n, rank, D = 3, 16, 1024
    c = _case(cuda, dtype, S, 2, 256, 256, D, n, rank, S, low=0.5)
    code, host = (z2.BF16, _bits) if dtype == "bf16" else (z2.F32, lambda t: t.cpu().numpy())
    gamma = np.random.default_rng(S).normal(1, 0.1, D).astype(np.float32) if weight else None
    ids = np.random.default_rng(S).integers(-1, n, S).astype(np.int32)
    ctx = z2.Context(0, S, 2, 256, D, 0, seed=1)
    ctx.set_adapters(host(c["A"]), host(c["B"]), 256, code, c["scale"].cpu().numpy())
    ctx.set_stream_adapters(ids)
    ctx.set_head(host(c["W"]), code, 256)
    ctx.set_out_norm(gamma, 1e-5)
    codes = torch.zeros((S, 2), dtype=torch.int32, device=cuda)
    logits = torch.zeros((S, 2, 256), device=cuda)
    ctx.step(c["h"], code, z2.SampleParams(0.7, 50, 0.9, 0.02, 1.0, 255), codes, logits_out=logits)
    torch.cuda.synchronize()
    h = c["h"].double().cpu().numpy()
    x = h / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(1e-5)))
    if weight:
        x = x * gamma.astype(np.float64)
    np_ = lambda t: t.double().cpu().numpy()
    ref, mag, low = R.head_adapters(np_(c["W"]), 256, 2, 256, x, np_(c["A"]), np_(c["B"]), ids, np_(c["scale"]), 15.0)
    half = 2.0 ** -8 if dtype == "bf16" else 16 * F   # f32: the normed rows' own roundings
    assert (np.abs(logits.cpu().numpy() - ref) <= _bound(c, ref, mag, low) + half * (mag + low)).all()
    # the adapters' part stands out of that bound, or the test would not see it missing
    bare = R.head_adapters(np_(c["W"]), 256, 2, 256, x, np_(c["A"]), np_(c["B"]), ids * 0 - 1, None, 15.0)[0]
    assert (np.abs(ref - bare) > _bound(c, ref, mag, low) + half * (mag + low)).any() or (ids < 0).all()
    assert z2.device_error() == 0
    ctx.close()


@pytest.mark.parametrize("S", [4, 150])
def test_context_calls_in_any_order(z2, cuda, S):
    """Norm, head and adapters set in either order and set again give the same bits; without norm and
    adapters they are those of a context that never had them; host and captured steps agree."""
    import torch
    n, rank, D, C, V = 3, 16, 512, 3, 256
    c = _case(cuda, "bf16", S, C, V, V, D, n, rank, S, low=0.3)
    W, A, B, sc = _bits(c["W"]), _bits(c["A"]), _bits(c["B"]), c["scale"].cpu().numpy()
    rs = np.random.default_rng(S)
    gamma, other = (rs.normal(1, 0.1, D).astype(np.float32) for _ in range(2))
    ids = rs.integers(-1, n, S).astype(np.int32)
    p = z2.SampleParams(0.7, 50, 0.9, 0.02, 1.0, V - 1)
    codes = torch.zeros((S, C), dtype=torch.int32, device=cuda)

    def logits(ctx):
        out = torch.zeros((S, C, V), device=cuda)
        ctx.step(c["h"], z2.BF16, p, codes, logits_out=out)
        torch.cuda.synchronize()
        return out

    def adapt(ctx, a=A):
        ctx.set_adapters(a, B, V, z2.BF16, sc)
        ctx.set_stream_adapters(ids)

    one, two, bare = (z2.Context(0, S, C, V, D, 0, seed=5) for _ in range(3))
    for ctx in (one, two, bare):
        ctx.set_head(W, z2.BF16, V)
    one.set_out_norm(gamma, 1e-5)
    adapt(one)
    adapt(two, A[::-1].copy())
    two.set_out_norm(other, 1e-5)
    logits(two)
    adapt(two)
    two.set_out_norm(gamma, 1e-5)
    two.set_head(W, z2.BF16, V)
    first = logits(one)
    assert torch.equal(first, logits(two))
    host = np.zeros((S, C), np.int32)
    one.set_rng(two.get_rng())
    one.step_host(_bits(c["h"]), z2.BF16, p, host)
    two.step(c["h"], z2.BF16, p, codes)
    torch.cuda.synchronize()
    assert np.array_equal(host, codes.cpu().numpy())
    graph, out = torch.cuda.CUDAGraph(), torch.zeros((S, C, V), device=cuda)
    with torch.cuda.graph(graph):
        one.step(c["h"], z2.BF16, p, codes, logits_out=out)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    one.set_out_norm(enable=False)
    one.set_stream_adapters(None)
    two.set_out_norm(enable=False)
    two.set_adapters(None, None, 0, z2.BF16)
    plain = logits(bare)
    assert torch.equal(plain, logits(two))
    # no row has an adapter: the adapters' GEMM, within the sums' roundings of the head's own
    c["ids"] = torch.full((S,), -1, dtype=torch.int32, device=cuda)
    _check(c, logits(one))
    assert z2.device_error() == 0
    for ctx in (one, two, bare):
        ctx.close()


def test_another_head_type_is_refused(z2, cuda):
    import torch
    c = _case(cuda, "bf16", 2, 2, 64, 64, 64, 2, 8, 1)
    ctx = z2.Context(0, 2, 2, 64, 64, 0, seed=1)
    ctx.set_head(c["W"].float().cpu().numpy(), z2.F32, 64)
    ctx.set_adapters(_bits(c["A"]), _bits(c["B"]), 64, z2.BF16)
    ctx.set_stream_adapters(np.zeros(2, np.int32))
    with pytest.raises(z2.Zonos2cuError) as e:
        ctx.step(c["h"].float(), z2.F32, z2.SampleParams(pad_id=63), torch.zeros((2, 2), dtype=torch.int32, device=cuda))
    assert e.value.code == z2.ESTATE
    for bad in ((c["A"][:, :, :32], c["B"]), (c["A"], c["B"][:1])):
        with pytest.raises(ValueError):
            ctx.set_adapters(_bits(bad[0].contiguous()), _bits(bad[1].contiguous()), 64, z2.BF16)
    ctx.close()


@pytest.mark.parametrize("S,D,dtype", [(1, 4, "bf16"), (24, 3, "bf16"), (150, 2, "bf16"), (3, 2, "f32")])
def test_a_speculative_step(z2, cuda, S, D, dtype):
    """The last block's tail, the head with each stream's adapter at every drafted position, and
    the check of the drafts, as one captured step over several turns: each stage against its
    formula on the values the one before gave it."""
    import torch
    C, V, dim, n, rank, H = 9, 1024, 512, 5, 16, 32
    rows = S * (D + 1)
    c = _case(cuda, dtype, rows, C, V, 1026, dim, n, rank, S)
    c["W"] = c["W"] * 3
    ids = torch.randint(-1, n, (S,), device=cuda, dtype=torch.int32)
    c["ids"] = ids.repeat_interleave(D + 1).contiguous()
    code = z2.BF16 if dtype == "bf16" else z2.F32
    t = c["h"].dtype
    resid, block, gate = (torch.empty(rows, dim, dtype=t, device=cuda) for _ in range(3))
    post, out_w = (torch.rand(dim, device=cuda) + 0.5 for _ in range(2))
    total, logits = torch.empty(rows, dim, dtype=t, device=cuda), torch.empty(rows, C, V, device=cuda)
    work = torch.empty(z2.head_adapters_work(code, rows, rank), dtype=torch.uint8, device=cuda)
    drafts = torch.empty(S, D, C, dtype=torch.int32, device=cuda)
    u = torch.empty(S, D + 1, C, 2, device=cuda)
    hist = torch.full((S, C, H), -1, dtype=torch.int32, device=cuda)
    at = torch.zeros(S, dtype=torch.int32, device=cuda)
    codes = torch.empty(S, D + 1, C, dtype=torch.int32, device=cuda)
    acc = torch.empty(S, dtype=torch.int32, device=cuda)
    p = z2.SampleParams(0.9, 60, 0.95, 0.01, 1.2, V - 1)

    def step():
        z2.block_norm(resid, block, total, c["h"], post_weight=post, gate=gate, gate_sigmoid=True, norm_weight=out_w)
        _call(z2, c, logits, work)
        z2.verify_drafts(logits.view(S, D + 1, C, V), p, drafts, u, codes, acc, hist=hist, hist_pos=at)

    g = torch.Generator(device=cuda)
    g.manual_seed(S)
    graph = torch.cuda.CUDAGraph()
    for x in (resid, block, gate):
        x.zero_()
    drafts.zero_(), u.zero_()
    with torch.cuda.graph(graph):
        step()
    hist.fill_(-1), at.zero_()
    for turn in range(4):
        for x in (resid, block, gate):
            x.copy_(torch.randn(rows, dim, generator=g, device=cuda))
        u.copy_(torch.rand(u.shape, generator=g, device=cuda))
        if turn % 2:   # the codes the target is surest of, by an earlier replay's logits
            ring, pos = hist.clone(), at.clone()
            graph.replay()
            hist.copy_(ring), at.copy_(pos)
            drafts.copy_(logits.view(S, D + 1, C, V)[:, :D].argmax(-1))
        else:
            drafts.copy_(torch.randint(0, V, drafts.shape, generator=g, device=cuda))
        ring, pos = hist.cpu().numpy(), at.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        np_ = lambda x: x.double().cpu().numpy()
        want = R.block_norm(np_(resid), np_(block), np_(post), 1e-5, np_(gate), True, 1.0, np_(out_w), 1e-5)
        half = 2.0 ** -8 if dtype == "bf16" else F
        assert (np.abs(np_(total) - want[0]) <= half * np.abs(want[0]) + 52 * F * (want[2] + np.abs(want[0]))).all()
        _check(c, logits, rows=sorted({0, rows // 2, rows - 1}))
        want = R.verify_drafts(logits.view(S, D + 1, C, V).cpu().numpy(), V, p, drafts.cpu().numpy(), u.cpu().numpy(),
                               None, None, ring, pos)
        for got, ref in zip((codes, acc, None, hist, at), want):
            assert got is None or np.array_equal(got.cpu().numpy(), ref)
    assert z2.device_error() == 0
