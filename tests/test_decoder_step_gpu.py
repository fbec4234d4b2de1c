"""The calls of a decoder's step together, as a server makes them: drafted tokens into the cache, their attention, the
block's tail, the 8-bit head, the drafts' check; then the sampler on the tokens that stand."""
import numpy as np
import pytest

import cache_ref as R

pytestmark = pytest.mark.gpu


def _norm(x, eps=1e-5):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("captured", [False, True])
def test_drafted_frames_through_a_block(z2, cuda, name, captured):
    import torch
    t = torch.bfloat16 if name == "bf16" else torch.float32
    g = torch.Generator().manual_seed(3)
    S, D, heads, kv, dim, page, n_cb, vocab = 5, 3, 8, 2, 64, 16, 3, 128
    wide, new = heads * dim, D + 1   # a drafted run and the token before it, for each stream
    rows = S * new
    cached = torch.tensor([0, 5, 40, 100, 17])
    pages = 12 * S
    dev = dict(device=cuda)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    k_pages, v_pages = (normal(pages, kv, page, dim).to(t).to(cuda) for _ in range(2))
    table = torch.randperm(pages, generator=g).view(S, 12).to(torch.int32).to(cuda)
    kv_len = (cached + new).to(torch.int32).to(cuda)
    q_start = (torch.arange(S + 1) * new).to(torch.int32).to(cuda)
    cache = z2.PagedCache(k_pages, v_pages, table, kv_len, q_start)
    hidden = normal(rows, wide).to(t).to(cuda)
    W_q, W_k, W_v = ((normal(wide, n) / wide ** 0.5).to(t).to(cuda) for n in (wide, kv * dim, kv * dim))
    gate = normal(rows, heads).to(t).to(cuda)
    freq = torch.tensor([10000.0 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32).to(cuda)
    W = normal(n_cb * (vocab + 2), wide) * 0.05
    head, head_scale = torch.empty(W.shape, dtype=torch.int8, **dev), torch.empty(len(W), **dev)
    z2.quantize_rows(W.to(cuda), head, head_scale)
    work = torch.empty(z2.head_i8_work(rows, wide), dtype=torch.uint8, **dev)
    q_out, mixed, resid, normed = (torch.zeros(rows, wide, dtype=t, **dev) for _ in range(4))
    logits = torch.zeros(S, new, n_cb, vocab, **dev)
    drafts = torch.randint(0, vocab, (S, D, n_cb), generator=g, dtype=torch.int32).to(cuda)
    uniforms = torch.rand(S, new, n_cb, 2, generator=g).to(cuda)
    codes, n_accepted = torch.zeros(S, new, n_cb, dtype=torch.int32, **dev), torch.zeros(S, dtype=torch.int32, **dev)
    knobs = z2.SampleParams(1.0, 20, 0.95, 0.0, 1.0, vocab - 1)
    q, k, v = hidden @ W_q, hidden @ W_k, hidden @ W_v

    def step():
        z2.cache_append(cache, q, k, v, q_out, freq=freq)
        z2.cache_attend(cache, q_out, mixed, gate=gate, max_new=new)
        z2.block_norm(hidden, mixed, resid, normed, post_eps=-1.0)
        z2.head_i8(head, head_scale, vocab + 2, n_cb, vocab, normed, logits, work)
        z2.verify_drafts(logits, knobs, drafts, uniforms, codes, n_accepted)

    if captured:
        before = k_pages.clone(), v_pages.clone()
        step()   # (set-up that may not be captured)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        k_pages.copy_(before[0])
        v_pages.copy_(before[1])
        for x in (q_out, mixed, resid, normed, logits, codes):
            x.zero_()
        graph.replay()
    else:
        step()
    torch.cuda.synchronize()
    assert z2.device_error() == 0

    # each call's own inputs through its definition
    host = R.Cache(k_pages, v_pages, table, kv_len, q_start)
    want, tol = R.attend(host, rows, q_out.cpu(), torch.zeros(rows, wide), gate=gate.cpu())
    assert bool(((mixed.cpu().double() - want).abs() <= tol).all())
    y, e = R.rotated(q[:new, :dim].cpu(), torch.arange(cached[0], cached[0] + new), None, 1e-5, freq.cpu(), False)
    assert bool(((q_out[:new, :dim].cpu().double() - y).abs() <= e + R.HALF[t] * (y.abs() + e)).all())
    r = hidden.double() + mixed.double()
    n = _norm(r)
    assert bool(((normed.double() - n).abs() <= 2 * R.HALF[t] * n.abs() + 1e-6).all())
    x = normed.double()
    most = x.abs().amax(1, keepdim=True)
    rounded = torch.round(127 * x / most)
    keep = torch.cat([torch.arange(c * (vocab + 2), c * (vocab + 2) + vocab) for c in range(n_cb)]).to(cuda)
    lg = (rounded @ head[keep].double().t()) * (most / 127) * head_scale[keep].double()
    lg = (15 * torch.tanh(lg / 15)).view(S, new, n_cb, vocab)
    assert bool(((logits.double() - lg).abs() <= 2.0 ** -20 * lg.abs() + 1e-12).all())
    # the 8-bit head against the unrounded one: half a step of either side in each product
    full = 15 * torch.tanh((x @ W.double().to(cuda)[keep].t()) / 15)
    assert float((lg.view(rows, -1) - full).norm() / full.norm()) < 0.02
    import operators_ref
    ref = operators_ref.verify_drafts(logits.cpu().numpy(), vocab, knobs, drafts.cpu().numpy(), uniforms.cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), ref[0]) and np.array_equal(n_accepted.cpu().numpy(), ref[1])

    # the tokens that do not stand leave: the lengths fall, and the next tokens are written over them
    kv_len.copy_(kv_len - new + n_accepted + 1 + 1)
    one = (torch.arange(S + 1)).to(torch.int32).to(cuda)
    q_start.copy_(one)
    z2.cache_append(cache, q[:S], k[:S], v[:S], q_out[:S], freq=freq)
    z2.cache_attend(cache, q_out[:S], mixed[:S], gate=gate[:S], max_new=1)
    host = R.Cache(k_pages, v_pages, table, kv_len, q_start)
    want, tol = R.attend(host, S, q_out[:S].cpu(), torch.zeros(S, wide), gate=gate[:S].cpu())
    assert bool(((mixed[:S].cpu().double() - want).abs() <= tol).all())
    z2.block_norm(hidden[:S], mixed[:S], resid[:S], normed[:S], post_eps=-1.0)
    one_step = torch.zeros(S, n_cb, vocab, **dev)
    z2.head_i8(head, head_scale, vocab + 2, n_cb, vocab, normed[:S], one_step, work)
    rng = torch.from_numpy(np.stack([z2.Xoshiro256(s).s for s in range(S)]).view(np.int64)).to(cuda)
    out = torch.zeros(S, n_cb, dtype=torch.int32, **dev)
    z2.sample_rows(one_step, z2.SampleParams(pad_id=vocab - 1), rng, out)
    assert bool(((out >= 0) & (out < vocab)).all())
