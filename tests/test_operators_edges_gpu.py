"""The adapters, the draft verification and the block tail together with other calls, past one tile
of work, and with values at the ends of their types."""
import threading

import numpy as np
import pytest

import operators_ref as R

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
