"""The adapters, the draft verification and the block tail together with other calls, past one tile
of work, and with values at the ends of their types."""
import threading

import numpy as np
import pytest

import operators_ref as R
from test_head_adapters_gpu import F, _call, _case, _check

pytestmark = pytest.mark.gpu


def test_verification_from_two_threads(z2, cuda):
    """Host threads with nine and two codebooks, each on a stream of its own, all at once."""
    import torch
    V, D, S, turns = 256, 2, 3, 2000
    p = z2.SampleParams(pad_id=V - 1)
    r = np.random.default_rng(4)
    jobs = []
    for C in (9, 2):
        s = dict(lg=r.normal(0, 3, (S, D + 1, C, V)).astype(np.float32), u=r.random((S, D + 1, C, 2), np.float32))
        s["t"] = s["lg"][:, :D].argmax(-1).astype(np.int32)
        d = {k: torch.from_numpy(v).to(cuda) for k, v in s.items()}
        codes = torch.zeros(S, D + 1, C, dtype=torch.int32, device=cuda)
        acc = torch.zeros(S, dtype=torch.int32, device=cuda)
        jobs.append((s, d, codes, acc, torch.cuda.Stream()))
    torch.cuda.synchronize()
    start, failed = threading.Barrier(2), []

    def work(job):
        _, d, codes, acc, stream = job
        try:
            start.wait()
            for _ in range(turns):
                z2.verify_drafts(d["lg"], p, d["t"], d["u"], codes, acc, stream=stream)
        except Exception as e:   # an exception of a thread would be lost
            failed.append(e)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for s, d, codes, acc, _ in jobs:
        want = R.verify_drafts(s["lg"], V, p, s["t"], s["u"])
        assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])


@pytest.mark.parametrize("batch,rank", [(3, 16), (3, 256), (70, 16), (300, 40), (600, 64), (5, 12)])
@pytest.mark.parametrize("t", [2.0 ** 128 - 2.0 ** 104, 2.0 ** 128])
def test_low_rank_products_at_the_end_of_f32(z2, cuda, batch, rank, t):
    """One row whose A h is the largest f32 (it rounds to infinity in bf16) or past it: its logits are
    the softcap, by B's sign; B times it; and nothing of it reaches the rows beside it."""
    import torch
    c = _case(cuda, "bf16", batch, 2, 130, 130, 128, 4, rank, batch)
    c["scale"][1] = 2 - 2.0 ** -23 if t < 2.0 ** 128 else 1.0
    row = batch // 2
    c["ids"][row] = 1
    c["A"][1, :, 5] = 0.0
    c["A"][1, 3, 5] = 2.0 ** 7 if t < 2.0 ** 128 else 2.0 ** 8
    c["W"][:, 5] = 0.0
    b = c["B"][1, :, 3].double().view(2, 130)
    assert (b != 0).all()
    rest = torch.arange(batch, device=cuda) != row
    clean, open_ = _call(z2, c), _call(z2, c, softcap=0.0)
    c["h"][row] = 0.0
    c["h"][row, 5] = 2.0 ** 120
    got = _call(z2, c)
    assert torch.equal(got[row].double(), 15.0 * b.sign()) and torch.equal(got[rest], clean[rest])
    got = _call(z2, c, softcap=0.0)
    if t < 2.0 ** 128:   # one product of three exact parts, then sums with zeros
        assert ((got[row].double() - b * t).abs() <= 8 * F * (b * t).abs()).all()
    else:
        assert torch.equal(got[row].double(), b.sign() * float("inf"))
    assert torch.equal(got[rest], open_[rest])
    assert z2.device_error() == 0


@pytest.mark.parametrize("n_cb", [65535, 65536])
def test_many_codebooks(z2, cuda, n_cb):
    """More codebooks than a launch grid has rows for."""
    c = _case(cuda, "bf16", 66, n_cb, 2, 2, 8, 2, 8, 1)
    _check(c, _call(z2, c))
    assert z2.device_error() == 0


def _exact(c, softcap=0.0):
    """The logits in 64 bits, on the GPU."""
    import torch
    h, (n, rank, _) = c["h"].double(), c["A"].shape
    keep = torch.cat([torch.arange(k * c["rows"], k * c["rows"] + c["vocab"], device=h.device) for k in range(c["n_cb"])])
    y = h @ c["W"][keep].double().t()
    for a in range(n):
        at = (c["ids"] == a).nonzero()[:, 0]
        if len(at):
            y[at] += c["scale"][a].double() * (h[at] @ c["A"][a].double().t()) @ c["B"][a][keep].double().t()
    return (softcap * torch.tanh(y / softcap) if softcap else y).view(len(h), c["n_cb"], c["vocab"])


# Relative error of the logits in the 2-norm.  The tensor cores cut off what an f32 accumulator
# does not hold: on average half a unit in the last place, which is ln 2 * 2^-24 of the
# accumulator, itself 2/3 of its last value on average over a random walk's steps.  A part of the head's depth is
# 48 steps: 1.32e-6.  A h: 16 steps of a warp at a depth of 2048 (32 at 4096), then additions of 8 warps
# and a multiplication; its three parts and 16 ranks at a time of B t: four more; rounded
# ones count 2^-24 / sqrt(3).
STEP = np.log(2.0) * 2.0 ** -24 * 2 / 3


def _low_rank(dim, rank):
    return dim // 128 * STEP + (4 + 10 + rank / 16) * F


# f32: four roundings in each sum of four products, of 1 to 4 of its terms' variance, then one of the
# result: sqrt(10 / 4 + 1) * 2^-24 / sqrt(3), once for W h and, in A h's place, again.
F32 = np.sqrt(3.5 / 3) * F


@pytest.mark.parametrize("dtype,batch,n_cb,vocab,rows,dim,n,rank", [
    ("bf16", 20, 12, 1024, 1024, 2048, 5, 16), ("bf16", 64, 13, 1000, 1002, 2048, 40, 24), ("bf16", 3, 40, 300, 301, 768, 2, 8),
    ("bf16", 20, 9, 1024, 1026, 4096, 5, 16), ("bf16", 700, 9, 1024, 1024, 2048, 6, 16), ("bf16", 1000, 9, 1000, 1001, 4096, 32, 40),
    ("bf16", 2500, 9, 1024, 1026, 1024, 100, 8), ("bf16", 130, 30, 700, 700, 2048, 3, 64), ("bf16", 21, 3, 500, 501, 2048, 4, 12),
    ("f32", 5, 9, 1024, 1026, 2048, 3, 12), ("f32", 21, 4, 333, 334, 2047, 3, 16)])
def test_precision_over_many_tiles(z2, cuda, dtype, batch, n_cb, vocab, rows, dim, n, rank):
    """Sizes at which an SM takes more than one tile, and depths of several parts; the adapters' share
    alone, so that W's does not hide it."""
    c = _case(cuda, dtype, batch, n_cb, vocab, rows, dim, n, rank, batch + n_cb, low=0.3)
    _check(c, _call(z2, c), rows=sorted({0, batch // 3, batch - 1}))
    bf16 = dtype == "bf16"
    low = _low_rank(dim, rank) if bf16 else 2 * F32
    if bf16 and rank % 8:   # additions in f32 that are rounded: a lane's chain of dim / 128 fours, five levels
        low = wide = (dim / 128 + 4 + 5) * F
    else:
        wide = min(dim // 16, 48) * STEP + 4 * F if bf16 else F32
    for share, tol in (("all", wide + low), ("adapters", low)):
        if share == "adapters":
            c["W"].zero_()
        got, want = _call(z2, c, softcap=0.0).double(), _exact(c)
        err, size = (got - want).norm(dim=(1, 2)), want.norm(dim=(1, 2))
        named = (c["ids"] >= 0) & (c["ids"] < n)
        assert named.any() and not named.all()
        assert (err <= tol * size).all(), (share, float((err / size.clamp(min=1e-30)).max()), tol)
        assert (share == "all") or (got[~named] == 0).all()
    assert z2.device_error() == 0


@pytest.mark.parametrize("dtype,batch", [("bf16", 5), ("bf16", 100), ("bf16", 520), ("f32", 6)])
def test_an_overflowing_row_reaches_no_other(z2, cuda, dtype, batch):
    """Products past f32 in one row leave the bits of the rows beside it."""
    import torch
    c = _case(cuda, dtype, batch, 2, 130, 130, 128, 4, 16, batch)
    for row in (0, batch // 2, batch - 1):
        clean = _call(z2, c)
        kept = c["h"][row].clone()
        rest = torch.arange(batch, device=cuda) != row
        for value in (3e38, float("inf"), float("nan")):
            c["h"][row] = value
            c["h"][row, ::2] *= -1
            assert torch.equal(_call(z2, c)[rest], clean[rest])
        c["h"][row] = kept


@pytest.mark.parametrize("dtype,rows", [("bf16", 4), ("bf16", 60), ("bf16", 200), ("bf16", 1500), ("f32", 4)])
def test_calls_behind_each_other(z2, cuda, dtype, rows):
    """Tail, head and verification launched without a pause, each turn on what the last one left in
    place: the bits of the same calls one at a time."""
    import torch
    C, V, dim, n, rank, D, turns = 2, 256, 512, 3, 16, 1, 12
    c = _case(cuda, dtype, rows, C, V, V, dim, n, rank, rows)
    code, S = (z2.BF16 if dtype == "bf16" else z2.F32), rows // (D + 1)
    start = [torch.randn(rows, dim, device=cuda).to(c["h"].dtype) for _ in range(2)]
    w = torch.rand(dim, device=cuda) + 0.5
    g = torch.Generator(device=cuda)
    g.manual_seed(rows)
    u = torch.rand(turns, S, D + 1, C, 2, generator=g, device=cuda)
    p = z2.SampleParams(0.9, 60, 0.95, 0.01, 1.2, V - 1)
    work = torch.empty(z2.head_adapters_work(code, rows, rank), dtype=torch.uint8, device=cuda)

    def go(wait):
        resid, block = (t.clone() for t in start)
        logits = torch.zeros(turns, rows, C, V, device=cuda)
        codes = torch.zeros(turns, S, D + 1, C, dtype=torch.int32, device=cuda)
        drafts = torch.zeros(S, D, C, dtype=torch.int32, device=cuda)
        acc = torch.zeros(S, dtype=torch.int32, device=cuda)
        hist = torch.full((S, C, 8), -1, dtype=torch.int32, device=cuda)
        at = torch.zeros(S, dtype=torch.int32, device=cuda)
        torch.cuda.synchronize()
        for k in range(turns):
            z2.block_norm(resid, block, resid, c["h"], scale=0.5, norm_weight=w)
            if wait:
                torch.cuda.synchronize()
            _call(z2, c, logits[k], work)
            if wait:
                torch.cuda.synchronize()
            z2.verify_drafts(logits[k].view(S, D + 1, C, V), p, drafts, u[k], codes[k], acc, hist=hist, hist_pos=at)
            if wait:
                torch.cuda.synchronize()
            # the tail again, over the rows that the head has just read
            z2.block_norm(c["h"], block, None, c["h"], post_eps=-1.0)
            z2.block_norm(resid, c["h"], None, block, gate=c["h"], gate_sigmoid=True)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return resid, block, logits, codes, acc, hist, at

    for a, b in zip(go(False), go(True)):
        assert torch.equal(a, b)
    assert z2.device_error() == 0


def _verified(z2, cuda, lg, t, u, p):
    import torch
    S, D1, C, V = lg.shape
    dev = [torch.from_numpy(np.ascontiguousarray(a)).to(cuda) for a in (lg, t, u)]
    codes = torch.zeros(S, D1, C, dtype=torch.int32, device=cuda)
    acc = torch.zeros(S, dtype=torch.int32, device=cuda)
    z2.verify_drafts(dev[0], p, dev[1], dev[2], codes, acc)
    torch.cuda.synchronize()
    want = R.verify_drafts(lg, V, p, t, u)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
    return acc.cpu().numpy()


NEAR = (0.0, 1e-8, 1e-7, 1e-6, 3e-6, 6e-6, 9e-6, 1.1e-5, 2e-5, 3e-5)


def _near_top_p(deep, temperature, spread, outside, V=1024, S=1500, top_p=0.9):
    """Logits whose mass ahead of token t is within a few 1e-6 of top_p, by more weight on the tokens
    behind the first one outside (they may overtake it) or less on those behind the last one inside."""
    r = np.random.default_rng(deep + int(10 * spread))
    lg = r.normal(0, spread, (S, V))
    lg[:, r.permutation(V)[:deep]] -= r.uniform(15, 110, deep)
    T, top_p = np.float64(np.float32(temperature)), np.float64(np.float32(top_p))
    t = np.zeros(S, np.int32)
    for i, row in enumerate(lg):
        order = np.argsort(-row, kind="stable")
        e = np.exp((row[order] - row[order[0]]) / T)
        before = np.cumsum(e) - e
        j = int(np.searchsorted(before, top_p * e.sum())) - (not outside)
        near = NEAR[i % len(NEAR)] * (1 if i // len(NEAR) % 2 else -1)
        more = before[j] / top_p / (1 + near) - e.sum()       # weight that the tail needs for it
        tail = order[j + 1:]
        row[tail] += T * np.log1p(more / e[j + 1:].sum())
        t[i] = order[j]
    return np.repeat(lg.astype(np.float32)[:, None, None], 2, 1), t[:, None, None], np.zeros((S, 2, 1, 2), np.float32)


@pytest.mark.parametrize("outside", [True, False])
@pytest.mark.parametrize("deep", [0, 400])
@pytest.mark.parametrize("temperature,spread", [(1.0, 0.5), (0.7, 1.0), (1.3, 0.0)])
def test_nuclei_that_end_at_the_drafted_code(z2, cuda, deep, temperature, spread, outside):
    """Nuclei of hundreds of tokens, the mass ahead of the drafted code within a few 1e-6 of top_p: f32
    may answer only what the definition in 64 bits does.  `deep` tokens lie far below the others."""
    p = z2.SampleParams(temperature, 0, 0.9, 0.0, 1.0, 1023)
    acc = _verified(z2, cuda, *_near_top_p(deep, temperature, spread, outside), p)
    assert outside or 0.2 < acc.mean() < 0.8


@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 0.95, 0.0), (50, 0.9, 0.02), (100, 1.0, 0.0), (0, 1.0, 0.05)])
def test_uniforms_next_to_the_drafted_codes_share(z2, cuda, top_k, top_p, min_p):
    """u0 within a few 1e-6 of p(t), and u1 of the residual's cumulative weights."""
    V, S = 1000, 1500
    p = z2.SampleParams(0.8, top_k, top_p, min_p, 1.0, V - 1)
    r = np.random.default_rng(top_k + int(100 * top_p))
    lg = r.normal(0, 0.4, (S, V)).astype(np.float32)
    t, u = np.zeros((S, 1, 1), np.int32), np.zeros((S, 2, 1, 2), np.float32)
    for i, row in enumerate(lg):
        tok, w, _ = R._distribution(row, np.zeros(V, bool), np.ones(V, bool), p)
        j = int(r.integers(0, len(tok)))
        t[i] = tok[j]
        near = 1 + NEAR[i % len(NEAR)] * (1 if i // len(NEAR) % 2 else -1)
        u[i, 0, 0, 0] = min(w[j] / w.sum() * near, 1 - 2.0 ** -24)
        left = np.where(tok == t[i, 0, 0], 0.0, w)
        for d, weights in ((0, left), (1, w)):
            if weights.sum() > 0:
                k = int(r.integers(0, len(tok)))
                u[i, d, 0, 1] = min(np.cumsum(weights)[k] / weights.sum() * near, 1 - 2.0 ** -24)
    acc = _verified(z2, cuda, np.repeat(lg[:, None, None], 2, 1), t, u, p)
    assert 0.2 < acc.mean() < 0.8


@pytest.mark.parametrize("batch,n,rank", [(5, 4096, 8), (300, 4096, 16), (2500, 4096, 16), (300, 4097, 16), (300, 3, 256),
                                          (2000, 7, 256)])
def test_many_adapters_and_ranks(z2, cuda, batch, n, rank):
    """The most adapters that the tensor-core kernels take and one more, and the most ranks."""
    c = _case(cuda, "bf16", batch, 1, 70, 70, 128, n, rank, batch + n)
    c["ids"][batch // 2], c["ids"][-1] = n - 1, n
    _check(c, _call(z2, c))
    assert z2.device_error() == 0


def test_the_most_drafts(z2, cuda):
    """4095 drafted frames that all stand but the last few, with the penalty's ring."""
    import torch
    V, D, C, H = 33, 4095, 1, 7
    r = np.random.default_rng(2)
    lg = r.normal(0, 1, (2, D + 1, C, V)).astype(np.float32)
    t = r.integers(0, V, (2, D, C)).astype(np.int32)
    np.put_along_axis(lg[:, :D], t[..., None].astype(np.int64), 40.0, -1)
    lg[1, D - 3] = 0.0
    u = r.random((2, D + 1, C, 2), np.float32)
    hist, at = r.integers(-1, V, (2, C, H)).astype(np.int32), np.array([3, 9], np.int32)
    p = z2.SampleParams(0.9, 10, 0.9, 0.0, 1.2, V - 1)
    d = [torch.from_numpy(a.copy()).to(cuda) for a in (lg, t, u, hist, at)]
    codes = torch.zeros(2, D + 1, C, dtype=torch.int32, device=cuda)
    acc = torch.zeros(2, dtype=torch.int32, device=cuda)
    z2.verify_drafts(d[0], p, d[1], d[2], codes, acc, hist=d[3], hist_pos=d[4])
    torch.cuda.synchronize()
    got = [x.cpu().numpy() for x in (codes, acc, d[3], d[4])]
    assert got[1][0] == D and got[1][1] in range(D - 3, D)
    # what was emitted are the drafts up to there, and the ring holds the last of the emitted frames
    for s in range(2):
        n = got[1][s]
        assert np.array_equal(got[0][s, :n], t[s, :n]) and (got[0][s, n + 1:] == -1).all()
        assert got[3][s] == (at[s] + n + 1) % H
        for k in range(n - H + 1, n + 1):
            assert got[2][s, 0, (at[s] + k) % H] == got[0][s, k, 0]


def test_past_32_bits_of_elements(z2, cuda):
    """Logits, hidden rows and tails of more than 2^31 elements: the last rows as in a call of their own."""
    import torch
    C, V, dim, n, rank = 9, 1024, 64, 5, 8
    rows = (1 << 31) // (C * V) + 2000
    c = _case(cuda, "bf16", 4000, C, V, V, dim, n, rank, 1)
    last = dict(c)
    c["h"] = c["h"].repeat((rows + 3999) // 4000, 1)[:rows].contiguous()
    c["ids"] = c["ids"].repeat((rows + 3999) // 4000)[:rows].contiguous()
    out = _call(z2, c)
    last["h"], last["ids"] = c["h"][-100:].clone(), c["ids"][-100:].clone()
    _check(last, out[-100:])
    _check(last, _call(z2, last))
    # the check of those logits, the last streams against a call of their own
    S, D = rows // 5, 4
    lg = out[:5 * S].view(S, D + 1, C, V)
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    t = torch.randint(0, V, (S, D, C), generator=g, device=cuda, dtype=torch.int32)
    t[::2] = lg[::2, :D].argmax(-1).int()
    u = torch.rand(S, D + 1, C, 2, generator=g, device=cuda)
    u[::2, ..., 0] *= 1e-3   # these drafts stand
    p = z2.SampleParams(pad_id=V - 1)

    def check(lg, t, u):
        codes = torch.zeros(len(lg), D + 1, C, dtype=torch.int32, device=cuda)
        acc = torch.zeros(len(lg), dtype=torch.int32, device=cuda)
        z2.verify_drafts(lg, p, t, u, codes, acc)
        return codes, acc

    whole, some = check(lg, t, u), check(lg[-50:].clone(), t[-50:], u[-50:])
    assert torch.equal(whole[0][-50:], some[0]) and torch.equal(whole[1][-50:], some[1])
    assert (some[1] == D).any() and (some[1] == 0).any()
    del out, lg
    for dim in (2048, 2047):
        m = (1 << 31) // dim + 100
        x = torch.zeros(m, dim, dtype=torch.bfloat16, device=cuda)
        x[-64:] = torch.randn(64, dim, generator=g, device=cuda).bfloat16()
        few = x[-64:].clone()
        z2.block_norm(x, x, x, None, scale=0.5)
        want = torch.empty_like(few)
        z2.block_norm(few, few, want, None, scale=0.5)
        assert torch.equal(x[-64:], want)
        del x
    torch.cuda.empty_cache()
