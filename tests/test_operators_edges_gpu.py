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
