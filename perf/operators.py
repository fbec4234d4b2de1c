"""Measured cases of three operators of the decode step, each in its plain form and as the library's call.

* ``adapt``  -- the output head beside low-rank adapters of many requests:
  ``cap * tanh((W h + s_a B_a (A_a h)) / cap)``, one adapter (or none) per hidden row;
* ``verify`` -- drafted frames checked against the sampler's distribution of the target's logits, from given
  random numbers: the longest accepted run of frames, then a corrected or a bonus frame;
* ``norm``   -- a block's output norm, gate, scaled residual sum and the norm that follows it.

``run(state)`` makes one pass: elementary torch operations where ``own`` is false, the library's entry points where
it is true.  ``exact`` gives the same from the definitions in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

CAP = 15.0
MASKED = -1e9   # a row without a logit at or above this is all masked
PAD = 1023

_lib = None


def _library():
    """The library's Python mirror, found beside this folder."""
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zonos2.cpp_b200"))
        import zonos2cu
        _lib = zonos2cu
    return _lib


def listed():
    head = dict(op="adapt", codebooks=9, vocab=1024, dim=2048)
    check = dict(op="verify", codebooks=9, vocab=1024, stride=1024, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02,
                 penalty=1.0, history=0, ragged=False, probs=True, allow=False, delay=-1)
    norm = dict(op="norm", dim=2048, gate="full", sigmoid=True, post=True, scale=0.5, pad=0)
    return [
        # one stream with its speaker's adapter: the latency of a single decode step
        dict(head, name="adapt-1", type="bf16", batch=1, rows=1024, adapters=8, rank=16),
        # a serving batch of 64 streams in arrival order, the head's rows as the checkpoint stores them
        dict(head, name="adapt-64", type="bf16", batch=64, rows=1026, adapters=16, rank=32),
        # guidance pairs or drafted positions of an odd number of streams
        dict(head, name="adapt-333", type="bf16", batch=333, rows=1024, adapters=24, rank=8),
        # one GPU's full batch of streams
        dict(head, name="adapt-4096", type="bf16", batch=4096, rows=1024, adapters=32, rank=16),
        # the 32-bit head of a few streams
        dict(head, name="adapt-f32-4", type="f32", batch=4, rows=1026, adapters=3, rank=12),
        # one stream, four drafted frames
        dict(check, name="verify-1", streams=1, drafts=4, agree=0.8),
        # a serving batch with its repetition history and streams that drafted less than the others
        dict(check, name="verify-64", streams=64, drafts=3, agree=0.8, penalty=1.2, history=256, ragged=True, stride=1026),
        # drafts looked up in the text so far (no draft distribution), no top-k, odd vocabulary
        dict(check, name="verify-lookup", streams=300, drafts=5, agree=0.7, probs=False, top_k=0, top_p=0.95, vocab=1001, stride=1001, temperature=1.0),
        # a full batch
        dict(check, name="verify-2048", streams=2048, drafts=4, agree=0.8, top_k=100, allow=True),
        # the last block's output of one stream
        dict(norm, name="norm-1", type="bf16", rows=1),
        # 32-bit rows with a gate per row, cut out of wider buffers
        dict(norm, name="norm-257-f32", type="f32", rows=257, gate="row", pad=64),
        # a prompt's worth of rows
        dict(norm, name="norm-16384", type="bf16", rows=16384),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["adapt", "verify", "norm"])
    if op == "adapt":
        f32 = rng.random() < 0.25
        vocab = rng.choice([1024, rng.randint(64, 1024)])
        return dict(op=op, type="f32" if f32 else "bf16", batch=_log(rng, 1, 12) if f32 else _log(rng, 1, 4096),
                    codebooks=rng.choice([9, rng.randint(1, 9)]), vocab=vocab, rows=vocab + rng.choice([0, 2]),
                    dim=rng.choice([2048, rng.randint(3, 256) if f32 else 8 * rng.randint(8, 256)]), adapters=_log(rng, 1, 64),
                    rank=rng.randint(1, 64) if f32 else 8 * rng.randint(1, 8))
    if op == "verify":
        vocab = rng.choice([1024, rng.randint(33, 1024)])
        penalty = rng.choice([1.0, rng.uniform(0.9, 1.4)])
        return dict(op=op, streams=_log(rng, 1, 1200), drafts=rng.randint(1, 6), agree=rng.uniform(0.2, 0.95), codebooks=rng.choice([9, rng.randint(1, 9)]),
                    vocab=vocab, stride=vocab + rng.choice([0, 2, 5]), temperature=rng.uniform(0.5, 1.3), top_k=rng.choice([0, 50, rng.randint(1, 200)]),
                    top_p=rng.choice([1.0, rng.uniform(0.5, 0.99)]), min_p=rng.choice([0.0, rng.uniform(0.01, 0.1)]), penalty=penalty,
                    history=0 if penalty == 1.0 else _log(rng, 2, 512), ragged=rng.random() < 0.5, probs=rng.random() < 0.7, allow=rng.random() < 0.4,
                    delay=rng.choice([-1, -1, rng.randint(0, 8)]))
    dim = rng.choice([2048, rng.randint(1, 64), rng.randint(65, 8192)])
    return dict(op=op, type=rng.choice(["bf16", "f32"]), rows=max(1, min(_log(rng, 1, 16384), (1 << 24) // dim)), dim=dim,
                gate=rng.choice(["full", "row", "dim", "none"]), sigmoid=rng.random() < 0.5, post=rng.random() < 0.7,
                scale=rng.uniform(0.1, 1.5), pad=rng.choice([0, 0, rng.randint(1, 40)]))


def _type(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def _float(x):
    """The value that a float knob has in 32 bits."""
    return float(np.float32(x))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "adapt":
        t, n, r, d = _type(case), case["adapters"], case["rank"], case["dim"]
        wide = case["codebooks"] * case["rows"]
        s["W"] = (normal(wide, d) * 0.02).to(t)
        s["hidden"] = normal(case["batch"], d).to(t)
        s["A"] = (normal(n, r, d) / math.sqrt(d)).to(t)
        s["B"] = (normal(n, wide, r) * 0.05).to(t)
        s["factor"] = 0.5 + 1.5 * uniform(n)
        s["which"] = whole(0, n, case["batch"])
        s["which"][uniform(case["batch"]) < 0.1] = -1   # streams without an adapter
        s["work"] = torch.empty(case["batch"] * r, dtype=torch.float64, device="cuda")
        s["out"] = torch.empty(case["batch"], case["codebooks"], case["vocab"], device="cuda")
        return s
    if case["op"] == "norm":
        t, n, d = _type(case), case["rows"], case["dim"]
        s["resid"] = (normal(n, d + case["pad"]) * 2).to(t)[:, :d]
        s["block"] = normal(n, d + case["pad"]).to(t)[:, :d]
        s["post_weight"], s["norm_weight"] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        shape = {"full": (n, d), "row": (n, 1), "dim": (1, d), "none": None}[case["gate"]]
        s["gate_values"] = normal(*shape).to(t).expand(n, d) if shape else None
        s["sum"], s["normed"] = torch.empty(n, d, dtype=t, device="cuda"), torch.empty(n, d, dtype=t, device="cuda")
        return s
    S, D, C, V, stride = case["streams"], case["drafts"], case["codebooks"], case["vocab"], case["stride"]
    full = torch.empty(S, D + 1, C, stride, device="cuda")
    full.copy_(CAP * torch.tanh(3.0 * normal(S, D + 1, C, stride) / CAP))
    logits = full[..., :V]
    good = uniform(S, D) < case["agree"]   # frames on which the draft and the target agree
    H = case["history"]
    s["ring"] = whole(-1, V, S, C, H) if H else None
    s["at"] = whole(0, H, S) if H else None
    s["bits"] = None
    may = torch.ones(S, 1, 1, V, dtype=torch.bool, device="cuda")
    if case["allow"]:
        words = (V + 31) // 32
        weights = torch.bitwise_left_shift(torch.ones(32, dtype=torch.int64, device="cuda"), torch.arange(32, device="cuda"))
        on = uniform(S, words, 32) < 0.9
        bits = (on.to(torch.int64) * weights).sum(-1)
        s["bits"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        may = on.view(S, 1, 1, -1)[..., :V]
    if case["probs"]:
        # the draft model: the target's logits with noise, under the same knobs; one token drawn from them
        noise = torch.where(good, 0.02, 1.5)[:, :, None, None]
        rough = logits[:, :D] + noise * normal(S, D, C, V)
        if H:
            tokens = torch.where(s["ring"] >= 0, s["ring"], V).long()
            seen = torch.zeros(S, C, V + 1, dtype=torch.bool, device="cuda").scatter_(-1, tokens, True)[:, None, :, :V]
            rough = torch.where(seen, torch.where(rough > 0, rough / case["penalty"], rough * case["penalty"]), rough)
        held = (case["delay"] + torch.arange(D, device="cuda"))[:, None] < torch.arange(C, device="cuda")
        if case["delay"] >= 0:
            may = torch.where(held[..., None], torch.arange(V, device="cuda") == min(PAD, V - 1), may)
        rough = rough.masked_fill(~may, -math.inf) / case["temperature"]
        q, rank = torch.softmax(rough, dim=-1).sort(-1, descending=True)
        if 0 < case["top_k"] < V:
            q[..., case["top_k"]:] = 0
        q = torch.where(q.cumsum(-1) - q < case["top_p"] * q.sum(-1, keepdim=True), q, 0.0)
        q = torch.where(q >= case["min_p"] * q[..., :1], q, 0.0)
        q /= q.sum(-1, keepdim=True)
        cdf = q.cumsum(-1)
        at = (cdf < uniform(S, D, C, 1) * cdf[..., -1:]).sum(-1, keepdim=True).clamp_(max=V - 1)
        draft = rank.gather(-1, at)[..., 0].to(torch.int32)
        s["q"] = torch.zeros_like(q).scatter_(-1, rank, q)
    else:
        # looked-up frames: where they are right the target is nearly sure of them
        draft = whole(0, V, S, D, C)
        spike = torch.where(good[..., None].expand(S, D, C), 14.9, -3.0)
        logits[:, :D].scatter_(-1, draft[..., None].long(), spike[..., None])
        s["q"] = None
    s["logits"], s["draft"] = full, draft
    s["count"] = whole(0, D + 1, S) if case["ragged"] else None
    s["u"] = uniform(S, D + 1, C, 2)
    s["codes"] = torch.empty(S, D + 1, C, dtype=torch.int32, device="cuda")
    s["flags"] = torch.empty(S, D + 1, C, dtype=torch.int32, device="cuda")
    s["accepted"] = torch.empty(S, dtype=torch.int32, device="cuda")
    return s


def _adapt(s):
    """The head in 32 bits: every adapter's projection, the rows' own ones kept, then both products summed."""
    n, r, C, V = s["adapters"], s["rank"], s["codebooks"], s["vocab"]
    h = s["hidden"].float()
    W = s["W"].float().view(C, s["rows"], -1)[:, :V].reshape(C * V, -1)
    B = s["B"].float().view(n, C, s["rows"], r)[:, :, :V].reshape(n, C * V, r)
    mine = (s["which"][:, None] == torch.arange(n, device=h.device)).float() * s["factor"]
    low = (h @ s["A"].float().view(n * r, -1).t()).view(-1, n, r) * mine[:, :, None]
    y = h @ W.t() + low.reshape(-1, n * r) @ B.permute(0, 2, 1).reshape(n * r, C * V)
    return (CAP * torch.tanh(y / CAP)).view(-1, C, V)


def _norm(s):
    r, y = s["resid"].float(), s["block"].float()
    if s["post"]:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * s["post_weight"]
    if s["gate_values"] is not None:
        g = s["gate_values"].float()
        y = y * (1 / (1 + torch.exp(-g)) if s["sigmoid"] else g)
    r = r + s["scale"] * y
    n = r / torch.sqrt((r * r).mean(-1, keepdim=True) + 1e-5) * s["norm_weight"]
    return r.to(_type(s)), n.to(_type(s))


def _verify(s):
    """The check in 64 bits (a code turns on a comparison, so values next to a border count)."""
    S, D, C, V, H = s["streams"], s["drafts"], s["codebooks"], s["vocab"], s["history"]
    dev = s["logits"].device
    x, draft = s["logits"][..., :V], s["draft"].long()
    place = torch.arange(D + 1, device=dev)
    odd = torch.isnan(x) | (x == math.inf)
    flags = odd.any(-1).int() * 2
    x = x.masked_fill(odd, -math.inf)
    if H:
        # the window at position d: the ring, its d oldest entries replaced by the frames drafted before
        age = (torch.arange(H, device=dev) - s["at"].long()[:, None]) % H                      # [S, H]
        last = age + torch.div(place[:, None, None] - 1 - age, H, rounding_mode="floor") * H   # [D+1, S, H]
        last = last.permute(1, 0, 2)[:, :, None, :].expand(S, D + 1, C, H)
        newer = draft.permute(0, 2, 1)[:, None].expand(S, D + 1, C, D).gather(-1, last.clamp(0, D - 1))
        seen = torch.where((age[:, None, None, :] < place[:, None, None]), newer, s["ring"].long()[:, None])
        seen = torch.where((seen >= 0) & (seen < V), seen, V)
        marks = torch.zeros(S, D + 1, C, V + 1, dtype=torch.bool, device=dev).scatter_(-1, seen, True)[..., :V]
        rho = _float(s["penalty"])
        x = torch.where(marks, torch.where(x > 0, x * _float(np.float32(1) / np.float32(rho)), x * rho), x)
    if s["bits"] is not None:
        may = (s["bits"][:, :, None] >> torch.arange(32, device=dev)) & 1
        x = x.masked_fill(may.view(S, 1, 1, -1)[..., :V] == 0, -math.inf)
    pad = min(PAD, V - 1)
    if s["delay"] >= 0:
        held = (s["delay"] + place)[:, None] < torch.arange(C, device=dev)
        x = x.masked_fill(held[..., None] & (torch.arange(V, device=dev) != pad), -math.inf)
    dead = x.max(-1).values < MASKED
    flags = flags | dead.int()
    x = torch.where(dead[..., None], torch.where(torch.arange(V, device=dev) == pad, 0.0, -math.inf), x)
    top, token = torch.sort(x, dim=-1, descending=True, stable=True)
    top = top.double()
    e = torch.exp((top - top[..., :1]) / _float(s["temperature"]))
    rank = torch.arange(V, device=dev)
    if 0 < s["top_k"] < V:
        e = torch.where(rank < s["top_k"], e, 0.0)
    if s["top_p"] < 1:
        before = e.cumsum(-1) - e
        e = torch.where((before < _float(s["top_p"]) * e.sum(-1, keepdim=True)) | (rank == 0), e, 0.0)
    if s["min_p"] > 0:
        e = torch.where(e >= _float(s["min_p"]), e, 0.0)
    p = e / e.sum(-1, keepdim=True)                                # by rank
    in_draft = p[:, :D].gather(-1, (token[:, :D] == draft[..., None]).int().argmax(-1, keepdim=True))[..., 0]
    if s["q"] is not None:
        q = s["q"].double()
        takes = s["u"][:, :D, :, 0].double() * q.gather(-1, draft[..., None])[..., 0] < in_draft
        q = q.gather(-1, token[:, :D])
    else:
        takes = s["u"][:, :D, :, 0].double() < in_draft
        q = (token[:, :D] == draft[..., None]).double()
    count = s["count"].long().clamp(0, D) if s["count"] is not None else torch.full((S,), D, device=dev)
    rest = p.clone()
    left = (p[:, :D] - q).clamp(min=0)
    drafted = (place[:D] < count[:, None])[:, :, None, None]
    rest[:, :D] = torch.where(drafted & (left.sum(-1, keepdim=True) > 0), left, p[:, :D])
    cum = rest.cumsum(-1)
    u = s["u"][..., 1:].double()
    hit = (cum >= u * cum[..., -1:]) & (rest > 0)
    some = hit.any(-1, keepdim=True)
    final = (rest > 0).int() * rank
    slot = torch.where(some, hit.int().argmax(-1, keepdim=True), final.argmax(-1, keepdim=True))
    drawn = token.gather(-1, slot)[..., 0]
    takes = takes & drafted[..., 0]
    n = takes.all(-1).int().cumprod(-1).sum(-1)
    code = drawn.clone()
    code[:, :D] = torch.where(takes, draft, drawn[:, :D])
    out = place > n[:, None]
    code = code.masked_fill(out[..., None], -1).int()
    flags = flags.masked_fill(out[..., None], 0).int()
    result = {"codes": code, "accepted": n.int(), "flags": flags}
    if H:
        slots = (s["at"].long()[:, None] + place) % H                                 # [S, D+1]
        keep = (place <= n[:, None]) & (place + H > n[:, None])                       # the last H frames
        where = torch.where(keep, slots, H)[:, None].expand(S, C, D + 1)
        wide = torch.cat([s["ring"], s["ring"][..., :1]], -1).scatter_(-1, where, code.permute(0, 2, 1))
        s["ring"].copy_(wide[..., :H])
        s["at"].copy_((s["at"] + n + 1) % H)
        result |= {"ring": s["ring"], "at": s["at"]}
    return result


def run(state):
    s = state
    if not own:
        return {"adapt": _adapt, "norm": _norm, "verify": _verify}[s["op"]](s)
    Z = _library()
    if s["op"] == "adapt":
        Z.head_adapters(s["W"], Z.BF16 if s["type"] == "bf16" else Z.F32, s["rows"], s["codebooks"], s["vocab"], s["hidden"],
                        s["A"], s["B"], s["which"], s["out"], s["work"], scale=s["factor"])
        return s["out"]
    if s["op"] == "norm":
        Z.block_norm(s["resid"], s["block"], s["sum"], s["normed"], post_weight=s["post_weight"] if s["post"] else None,
                     post_eps=1e-5 if s["post"] else -1.0, gate=s["gate_values"], gate_sigmoid=s["sigmoid"], scale=s["scale"],
                     norm_weight=s["norm_weight"], norm_eps=1e-5)
        return s["sum"], s["normed"]
    knobs = Z.SampleParams(s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["penalty"], min(PAD, s["vocab"] - 1))
    Z.verify_drafts(s["logits"], knobs, s["draft"], s["u"], s["codes"], s["accepted"], vocab=s["vocab"], draft_probs=s["q"], n_drafts=s["count"],
                    flags=s["flags"], hist=s["ring"], hist_pos=s["at"], allow=s["bits"], delay_step=s["delay"])
    result = {"codes": s["codes"], "accepted": s["accepted"], "flags": s["flags"]}
    if s["history"]:
        result |= {"ring": s["ring"], "at": s["at"]}
    return result


def work(case):
    if case["op"] == "adapt":
        size = 2 if case["type"] == "bf16" else 4
        b, r, d, n = case["batch"], case["rank"], case["dim"], case["codebooks"] * case["vocab"]
        used = case["adapters"] * (1 - (1 - 0.9 / case["adapters"]) ** b)   # adapters that some row has
        return {"bytes": size * (n * d + b * d + used * r * (d + n)) + 4 * b * n, "flops": 2 * b * (n * d + 0.9 * r * (d + n))}
    if case["op"] == "norm":
        size = 2 if case["type"] == "bf16" else 4
        gate = {"full": case["rows"] * case["dim"], "row": case["rows"], "dim": case["dim"], "none": 0}[case["gate"]]
        return {"bytes": size * (4 * case["rows"] * case["dim"] + gate) + 8 * case["dim"], "flops": 10 * case["rows"] * case["dim"]}
    # a stream's frames are needed up to the first that is not accepted (about the share `agree` of them is), half as many drafted where ragged
    S, D, C, V = case["streams"], case["drafts"], case["codebooks"], case["vocab"]
    drafted = D / 2 if case["ragged"] else D
    frames = sum(case["agree"] ** d for d in range(int(drafted) + 1)) + (drafted % 1) * case["agree"] ** (int(drafted) + 1)
    q = (4 * V * min(1, frames * (1 - case["agree"])) if case["probs"] else 0) + 4 * frames   # one frame's codes are corrected
    return {"bytes": S * C * (4 * V * frames + q + 12 * frames + 8 * (D + 1) + (4 * case["history"])) + (S * V / 8 if case["allow"] else 0),
            "flops": S * C * frames * V * 6}


def _exact_row(x, marks, may, forced, case, pad):
    """(tokens in order, probabilities, flag) of one row in 64 bits."""
    x = x.astype(np.float32).copy()
    bad = np.isnan(x) | (x == np.inf)
    flag = 2 if bad.any() else 0
    x[bad] = -np.inf
    if marks is not None:
        rho = np.float32(case["penalty"])
        m = np.flatnonzero(marks)
        x[m] = np.where(x[m] > 0, x[m] * (np.float32(1) / rho), x[m] * rho)
    if may is not None:
        x[~may] = -np.inf
    if forced:
        x[np.arange(x.size) != pad] = -np.inf
    if not x.max() >= MASKED:
        return np.array([pad]), np.array([1.0]), flag | 1
    k = case["top_k"] if 0 < case["top_k"] < x.size else x.size
    order = np.lexsort((np.arange(x.size), -x.astype(np.float64)))[:k]
    e = np.exp((x[order].astype(np.float64) - float(x.max())) / _float(case["temperature"]))
    if case["top_p"] < 1:
        keep = int(np.searchsorted(np.cumsum(e), _float(case["top_p"]) * math.fsum(e), side="left")) + 1
        order, e = order[:keep], e[:keep]
    if case["min_p"] > 0:
        keep = max(1, int((e >= _float(case["min_p"])).sum()))
        order, e = order[:keep], e[:keep]
    return order, e / math.fsum(e), flag


def _exact_verify(case, seed):
    s = prepare(case, seed)
    take = lambda name: None if s[name] is None else s[name].cpu().numpy()  # noqa: E731
    logits, draft, u, q, count, ring, at, bits = (take(n) for n in ("logits", "draft", "u", "q", "count", "ring", "at", "bits"))
    S, D, C, V, H = case["streams"], case["drafts"], case["codebooks"], case["vocab"], case["history"]
    pad = min(PAD, V - 1)
    codes, flags, accepted = np.full((S, D + 1, C), -1, np.int32), np.zeros((S, D + 1, C), np.int32), np.zeros(S, np.int32)
    for i in range(S):
        many = D if count is None else min(max(int(count[i]), 0), D)
        may = None
        if bits is not None:
            may = np.unpackbits(bits[i].view(np.uint8), bitorder="little")[:V].astype(bool)
        window = None if H == 0 else ring[i].copy()
        for d in range(many + 1):
            every = True
            for c in range(C):
                marks = None
                if H:
                    marks = np.zeros(V, bool)
                    got = window[c][(window[c] >= 0) & (window[c] < V)]
                    marks[got] = True
                order, p, flags[i, d, c] = _exact_row(logits[i, d, c, :V], marks, may, case["delay"] >= 0 and case["delay"] + d < c, case, pad)
                w = p
                if d < many:
                    t = int(draft[i, d, c])
                    here = np.flatnonzero(order == t)
                    chance = float(p[here[0]]) if here.size else 0.0
                    of_t = 1.0 if q is None else float(q[i, d, c, t])
                    if float(u[i, d, c, 0]) * of_t < chance:
                        codes[i, d, c] = t
                        continue
                    every = False
                    other = (order == t).astype(np.float64) if q is None else q[i, d, c][order].astype(np.float64)
                    left = np.maximum(p - other, 0)
                    w = left if left.sum() > 0 else p
                run_sum = np.cumsum(w)
                ok = np.flatnonzero((run_sum >= float(u[i, d, c, 1]) * run_sum[-1]) & (w > 0))
                codes[i, d, c] = order[ok[0]] if ok.size else order[np.flatnonzero(w > 0)[-1]]
            if H:
                window[:, (int(at[i]) + d) % H] = codes[i, d]
            if d == many or not every:
                accepted[i] = d
                break
        if H:
            ring[i] = window
            at[i] = (int(at[i]) + int(accepted[i]) + 1) % H
    result = {"codes": codes, "accepted": accepted, "flags": flags}
    return result | {"ring": ring, "at": at} if H else result


def exact(case, seed):
    if case["op"] == "verify":
        return _exact_verify(case, seed)
    s = prepare(case, seed)
    if case["op"] == "norm":
        r, y = s["resid"].double(), s["block"].double()
        if case["post"]:
            y = y * (y.pow(2).sum(1) / case["dim"] + _float(1e-5)).pow(-0.5)[:, None] * s["post_weight"].double()
        if s["gate_values"] is not None:
            y = y * (torch.sigmoid(s["gate_values"].double()) if case["sigmoid"] else s["gate_values"].double())
        r = torch.add(r, y, alpha=_float(case["scale"]))
        n = r * (r.pow(2).sum(1) / case["dim"] + _float(1e-5)).pow(-0.5)[:, None] * s["norm_weight"].double()
        return r, n
    C, V, rows = case["codebooks"], case["vocab"], case["rows"]
    keep = torch.cat([torch.arange(c * rows, c * rows + V, device="cuda") for c in range(C)])
    h = s["hidden"].double()
    y = torch.mm(h, s["W"][keep].double().t())
    for a in range(case["adapters"]):
        at = torch.nonzero(s["which"] == a)[:, 0]
        if at.numel():
            y[at] += s["factor"][a].double() * torch.mm(torch.mm(h[at], s["A"][a].double().t()), s["B"][a][keep].double().t())
    return (CAP * torch.tanh(y / CAP)).view(-1, C, V)
