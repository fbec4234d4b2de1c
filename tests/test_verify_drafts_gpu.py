"""Draft verification against its definition in 64 bits: every code, flag and ring equal."""
import numpy as np
import pytest

import operators_ref as R

pytestmark = pytest.mark.gpu


def _case(S, D, C, V, seed, spread=3.0, stride=None, certain=False, H=0, ragged=False, allow=None, near=0.05):
    r = np.random.default_rng(seed)
    lg = np.zeros((S, D + 1, C, stride or V), np.float32)
    lg[:] = np.nan   # what lies past the vocabulary is not read as a logit
    lg[..., :V] = r.normal(0, spread, (S, D + 1, C, V))
    s = dict(logits=lg, u=r.random((S, D + 1, C, 2), np.float32))
    rough = lg[:, :D, :, :V] + r.normal(0, near, (S, D, C, V))
    q = np.exp(rough - rough.max(-1, keepdims=True)) if D else np.zeros((S, 0, C, V))
    q = q / q.sum(-1, keepdims=True) if D else q
    at = (q.cumsum(-1) < r.random((S, D, C, 1))).sum(-1).clip(0, V - 1)
    s["drafts"] = at.astype(np.int32)
    s["probs"] = None if certain else q.astype(np.float32)
    s["n_drafts"] = r.integers(-1, D + 2, S).astype(np.int32) if ragged else None
    s["hist"] = r.integers(-1, V, (S, C, H)).astype(np.int32) if H else None
    s["hist_pos"] = r.integers(-3, 3 * H, S).astype(np.int32) if H else None
    words = (V + 31) // 32
    s["allow"] = (r.random((S, words, 32)) < allow).astype(np.uint32) if allow else None
    if allow:
        bits = s["allow"] << np.arange(32, dtype=np.uint32)
        s["allow"] = np.bitwise_or.reduce(bits, -1).astype(np.uint32).view(np.int32)
    return s


def _run(z2, cuda, s, p, V, delay=-1, stream=None, flags=True):
    import torch
    d = {k: None if v is None else torch.from_numpy(v.copy()).to(cuda) for k, v in s.items()}
    S, D1, C, _ = s["logits"].shape
    codes, fl = (torch.full((S, D1, C), 99, dtype=torch.int32, device=cuda) for _ in range(2))
    acc = torch.full((S,), 99, dtype=torch.int32, device=cuda)
    z2.verify_drafts(d["logits"], p, d["drafts"], d["u"], codes, acc, vocab=V, draft_probs=d["probs"],
                     n_drafts=d["n_drafts"], flags=fl if flags else None, hist=d["hist"],
                     hist_pos=d["hist_pos"], allow=d["allow"], delay_step=delay, stream=stream)
    torch.cuda.synchronize()
    got = dict(codes=codes, accepted=acc, hist=d["hist"], hist_pos=d["hist_pos"])
    if flags:
        got["flags"] = fl
    return {k: None if v is None else v.cpu().numpy() for k, v in got.items()}


def _compare(z2, cuda, s, p, V, delay=-1, flags=True, stream=None):
    with np.errstate(all="ignore"):
        names = ("codes", "accepted", "flags", "hist", "hist_pos")
        want = dict(zip(names, R.verify_drafts(s["logits"], V, p, s["drafts"], s["u"], s["probs"], s["n_drafts"],
                                               s["hist"], s["hist_pos"], s["allow"], delay)))
    got = _run(z2, cuda, s, p, V, delay, stream, flags)
    for k, v in got.items():
        assert (v is None) == (want[k] is None)
        assert v is None or np.array_equal(v, want[k]), k
    return got


def _p(z2, V, **kw):
    a = dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.02, repetition_penalty=1.0, pad_id=V - 1)
    a.update(kw)
    return z2.SampleParams(**a)


@pytest.mark.parametrize("S,D,C,V,stride", [
    (1, 0, 1, 1, None), (1, 4, 9, 1024, None), (2, 3, 9, 1024, 1026), (3, 12, 2, 1001, 1003), (1, 9, 16, 33, 36),
    (5, 1, 9, 5, None), (40, 5, 9, 1000, None), (160, 2, 9, 64, None), (330, 2, 9, 1024, 1025), (2, 20, 3, 77, 80)])
def test_shapes(z2, cuda, S, D, C, V, stride):
    """One block and a cluster per stream, more positions than a cluster holds, 16 codebooks,
    unaligned rows, tiny vocabularies, no drafts at all."""
    s = _case(S, D, C, V, S + D + V, stride=stride, near=0.01)
    _compare(z2, cuda, s, _p(z2, V), V)


@pytest.mark.parametrize("S,D,C,V", [(1, 4, 2, 1024), (3, 12, 1, 300), (1, 30, 1, 1001), (300, 9, 2, 64)])
@pytest.mark.parametrize("near", [0.0, 0.01])
def test_long_runs(z2, cuda, S, D, C, V, near):
    """Drafts from the target's own distribution: many stand, over several rounds of a cluster."""
    s = _case(S, D, C, V, S + D, near=near)
    got = _compare(z2, cuda, s, _p(z2, V, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), V)
    # a code is refused with probability sum |p - q| / 2 < near, and by rounding of q
    assert got["accepted"].mean() > 0.5 * D


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("spread", [0.0, 0.3, 1.5, 4.0])
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (0, 0.95, 0.0), (0, 1.0, 0.05), (1, 0.9, 0.0),
                                               (50, 0.9, 0.02), (100, 1.0, 0.0), (150, 0.8, 0.0), (200, 0.99, 0.1),
                                               (700, 0.5, 0.0), (0, 0.0, 0.0), (20, 0.3, 1.0), (5000, 0.999999, 1e-6)])
def test_cuts(z2, cuda, certain, spread, top_k, top_p, min_p):
    """Lists that 128 candidates hold, that 256 hold, and that only the whole row holds; ties
    throughout (spread 0)."""
    V = 1024
    s = _case(6, 2, 9, V, 7, spread=spread, certain=certain)
    if certain:   # half of them at the largest logit
        top = s["logits"][:, :2].argmax(-1).astype(np.int32)
        s["drafts"] = np.where(s["u"][:, :2, :, 1] < 0.5, top, s["drafts"])
    _compare(z2, cuda, s, _p(z2, V, top_k=top_k, top_p=top_p, min_p=min_p), V)


@pytest.mark.parametrize("H", [1, 3, 64])
@pytest.mark.parametrize("rho", [0.7, 1.3])
@pytest.mark.parametrize("S", [2, 200])
def test_penalty_and_ring(z2, cuda, H, rho, S):
    """Rings shorter than the drafts, positions out of range, ragged drafts, and the ring after."""
    s = _case(S, 5, 4, 100, 31 + H, H=H, ragged=True, near=0.02)
    _compare(z2, cuda, s, _p(z2, 100, repetition_penalty=rho, top_k=0, top_p=0.98), 100)


def test_ring_without_penalty(z2, cuda):
    s = _case(3, 4, 2, 50, 12, H=7, near=0.0)
    _compare(z2, cuda, s, _p(z2, 50), 50)


@pytest.mark.parametrize("delay", [-1, 0, 4])
@pytest.mark.parametrize("V", [33, 1024])
def test_masks(z2, cuda, delay, V):
    """Allowed tokens and the delay pattern, a stream that allows nothing among them."""
    s = _case(8, 3, 9, V, 3 + V, allow=0.6)
    s["allow"][2] = 0
    s["drafts"][3, 0] = V - 1
    got = _compare(z2, cuda, s, _p(z2, V), V, delay, flags=True)
    assert (got["flags"][2, 0] == 1).all() and (got["codes"][2, 0] == V - 1).all()
    _compare(z2, cuda, s, _p(z2, V), V, delay, flags=False)


def test_odd_values(z2, cuda):
    """NaN and infinities among the logits, rows without any, logits at the ends of f32, drafts
    outside the vocabulary, and draft probabilities that are no distribution."""
    V, inf = 200, np.inf
    s = _case(24, 2, 3, V, 77)
    lg, q, u, t = s["logits"], s["probs"], s["u"], s["drafts"]
    lg[0, 0, 0, 5] = np.nan
    lg[1, 0, 1, 7] = inf
    lg[2, 0, 2, :] = -inf
    lg[3, 0, 0, :] = np.nan
    lg[4, 0] = -2e9
    lg[5, 0, 0, 3:] = -inf
    lg[6, 0] *= 1e30
    lg[7, 0, 1, 9] = 3.4e38
    lg[8, 0, 1, :] = -3.4e38
    lg[8, 0, 1, 3] = 0.0
    t[9, 0, 0], t[9, 1, 1], t[10, 0, 2] = -1, V, 1 << 30
    q[11, 0, 0, :] = 0.0
    q[12, 0, 1, :] = np.nan
    q[13, 0, 2, t[13, 0, 2]] = inf
    q[14, 0, 0, :] = 1.0
    q[15, 0, 0, :] = -1.0
    u[16:18] = 0.0
    u[18:20] = np.float32(1 - 2.0 ** -24)
    u[20, :, :, 1] = 0.0
    t[4, 0] = V - 1
    for p in (_p(z2, V), _p(z2, V, top_k=0, top_p=1.0, min_p=0.0), _p(z2, V, top_k=0, top_p=0.9, temperature=1e-3),
              _p(z2, V, temperature=1e4, top_k=0, top_p=0.5), _p(z2, V, temperature=1e-30),
              _p(z2, V, temperature=1e30)):
        _compare(z2, cuda, s, p, V)


def test_distribution(z2, cuda):
    """Drafts drawn from another distribution leave the emitted frame the target's: 40000 streams
    of one row, each frequency within 5 deviations of its probability."""
    V, S = 12, 40000
    r = np.random.default_rng(8)
    lg = r.normal(0, 1, V).astype(np.float32)
    q = r.dirichlet(np.ones(V)).astype(np.float32)
    s = dict(logits=np.tile(lg, (S, 2, 1, 1)), u=r.random((S, 2, 1, 2), np.float32),
             drafts=r.choice(V, (S, 1, 1), p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int32),
             probs=np.tile(q, (S, 1, 1, 1)), n_drafts=None, hist=None, hist_pos=None, allow=None)
    p = _p(z2, V, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    got = _run(z2, cuda, s, p, V)
    want = np.exp(lg.astype(np.float64))
    want /= want.sum()
    freq = np.bincount(got["codes"][:, 0, 0], minlength=V) / S
    assert (np.abs(freq - want) <= 5 * np.sqrt(want * (1 - want) / S)).all()
    accept = np.minimum(want, q.astype(np.float64)).sum()
    assert abs(got["accepted"].mean() - accept) <= 5 * np.sqrt(accept * (1 - accept) / S)


def test_captured_steps(z2, cuda):
    """A step recorded once and replayed: the ring it leaves is what the next one reads."""
    import torch
    V, S, D, C, H = 128, 20, 3, 9, 16
    cases = [_case(S, D, C, V, 50 + i, H=H, near=0.02) for i in range(4)]
    p = _p(z2, V, repetition_penalty=1.2)
    ring, at = cases[0]["hist"], cases[0]["hist_pos"]
    d = {k: torch.from_numpy(v.copy()).to(cuda) for k, v in cases[0].items() if v is not None}
    codes = torch.empty(S, D + 1, C, dtype=torch.int32, device=cuda)
    acc = torch.empty(S, dtype=torch.int32, device=cuda)

    def call():
        z2.verify_drafts(d["logits"], p, d["drafts"], d["u"], codes, acc, draft_probs=d["probs"],
                         hist=d["hist"], hist_pos=d["hist_pos"])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for c in cases:
        for k in ("logits", "drafts", "u", "probs"):
            d[k].copy_(torch.from_numpy(c[k]))
        graph.replay()
        want = R.verify_drafts(c["logits"], V, p, c["drafts"], c["u"], c["probs"], None, ring, at)
        ring, at = want[3], want[4]
        assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
        assert np.array_equal(d["hist"].cpu().numpy(), ring) and np.array_equal(d["hist_pos"].cpu().numpy(), at)


def test_other_stream(z2, cuda):
    import torch
    s = _case(4, 3, 9, 1024, 5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _compare(z2, cuda, s, _p(z2, 1024), 1024, stream=side)


@pytest.mark.parametrize("temperature", [0.7, 0.83, 1.1])
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 0.9, 0.0), (7, 0.97, 0.0), (0, 1.0, 0.05), (3, 0.9, 0.0)])
def test_lists_that_end_on_a_bucket_edge(z2, cuda, temperature, top_k, top_p, min_p):
    """The kernel sorts logits into buckets of an eighth of the temperature: lists whose last logit lies
    on a bucket's rounded edge, a few steps of f32 to either side."""
    V, S, m = 64, 6000, 6
    r = np.random.default_rng(int(temperature * 100) + top_k)
    s = _case(S, 0, 1, V, 3, certain=True)
    scale = np.float32(8) * np.float32(1.0 / np.float64(np.float32(temperature)))
    lg = np.full((S, V), -np.inf, np.float32)
    for row in lg:
        top = np.float32(r.uniform(-6, 6))
        low = np.float32(np.float64(top) - (r.integers(0, 60) + 0.5) / np.float64(scale))
        for _ in range(abs(k := int(r.integers(-2, 3)))):
            low = np.nextafter(low, np.float32(np.copysign(np.inf, k)))
        at = r.permutation(V)[:m]
        row[at] = r.uniform(low, top, m)
        row[at[:2]] = top, low
    s["logits"][:, 0, 0] = lg
    _compare(z2, cuda, s, _p(z2, V, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p), V)
