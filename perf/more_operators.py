"""Measured cases of three operators of a decoder that serves many streams, each in its plain form and as the library's call.

* ``append`` -- new tokens' queries and keys normalised per head and rotated by their positions, keys and values
  written to the streams' pages of a paged cache;
* ``attend`` -- the new tokens' attention over the pages: one token, a drafted run or a prompt's chunk per stream,
  causal, with grouped heads, an optional window and a gate per head;
* ``head8``  -- the output head in 8-bit integers, hidden rows rounded on the way with a scale for each, the
  weights with a scale for each row: ``cap * tanh(s_b s_n (q_b . w_n) / cap)``.

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
EPS = 1e-5
THETA = 10000.0

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
    cache = dict(type="bf16", heads=16, kv_heads=4, dim=128, page=16, ragged=False, pad=0)
    append = dict(cache, op="append", rot=128, halves=False, norm=True)
    attend = dict(cache, op="attend", window=0, gate=True)
    head = dict(op="head8", type="bf16", codebooks=9, vocab=1024, rows=1024, dim=2048)
    return [
        # one stream's next token
        dict(append, name="append-1", streams=1, new=1, least=6000, most=6144),
        # a serving batch with drafted frames, streams that drafted less than the others, rows cut out of wider buffers
        dict(append, name="append-64", streams=64, new=5, least=64, most=6144, ragged=True, pad=128),
        # prompts
        dict(append, name="append-prompt", streams=16, new=1024, least=0, most=2048, page=64, ragged=True),
        # one stream's next token, most of the longest sequence behind it
        dict(attend, name="attend-1", streams=1, new=1, least=6000, most=6144),
        # a serving batch with drafted frames
        dict(attend, name="attend-64", streams=64, new=5, least=64, most=6144, ragged=True),
        # a full batch, one token each
        dict(attend, name="attend-256", streams=256, new=1, least=256, most=4096, page=64),
        # long prompts in chunks, part of each already cached
        dict(attend, name="attend-prompt", streams=4, new=2048, least=2048, most=4096, page=64),
        # 32-bit chunks over the last tokens only, an odd number of them, rows cut out of wider buffers
        dict(attend, name="attend-f32", type="f32", streams=6, new=333, least=100, most=2000, page=32, ragged=True, window=512, pad=64),
        # one stream: the latency of a single decode step
        dict(head, name="head8-1", batch=1),
        # a serving batch, the head's rows as the checkpoint stores them
        dict(head, name="head8-64", batch=64, rows=1026),
        # drafted positions of an odd number of streams, 32-bit hidden rows
        dict(head, name="head8-333", type="f32", batch=333),
        # one GPU's full batch of streams
        dict(head, name="head8-4096", batch=4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "head8"])
    if op == "head8":
        vocab = rng.choice([1024, rng.randint(33, 1024)])
        return dict(op=op, type=rng.choice(["bf16", "bf16", "f32"]), batch=_log(rng, 1, 4096), codebooks=rng.choice([9, rng.randint(1, 9)]),
                    vocab=vocab, rows=vocab + rng.choice([0, 2]), dim=rng.choice([2048, 16 * rng.randint(1, 128)]))
    kind = rng.choice(["bf16", "bf16", "f32"])
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8, rng.randint(1, 8)])
    while kv * group > 16:
        kv //= 2
    dim = rng.choice([64, 128, 8 * rng.randint(2, 32)])
    kv = min(kv, max(1, 512 // dim))
    new = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 2048)])
    most = _log(rng, 16, 4096)
    streams = _log(rng, 1, 256)
    # no more tokens, cached tokens or scores than the largest listed ones have
    streams = max(1, min(streams, 8192 // new, (1 << 19) // (most + new), (1 << 25) // (new * (most + new))))
    if kind == "f32" or dim > 128:
        streams = max(1, min(streams, (1 << 18) // (most + new), (1 << 21) // (new * (most + new))))
    case = dict(op=op, type=kind, streams=streams, new=new, least=rng.choice([0, most // 2, most]), most=most, heads=kv * group, kv_heads=kv, dim=dim,
                page=rng.choice([8, 16, 32, 64, 128, 256]), ragged=rng.random() < 0.7, pad=rng.choice([0, 0, 8 * rng.randint(1, 8)]))
    if op == "append":
        return case | dict(rot=rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)]), halves=rng.random() < 0.5, norm=rng.random() < 0.7)
    return case | dict(window=rng.choice([0, 0, _log(rng, 1, 1024)]), gate=rng.random() < 0.5)


def _type(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    t = _type(case)
    if case["op"] == "head8":
        wide = case["codebooks"] * case["rows"]
        w = normal(wide, case["dim"]) * 0.02
        most = w.abs().amax(1, keepdim=True)
        s["W"] = torch.round(w * 127 / most).to(torch.int8)
        s["w_scale"] = (most[:, 0] / 127).contiguous()
        s["hidden"] = (normal(case["batch"], case["dim"]) * (0.5 + normal(case["batch"], 1).abs())).to(t)
        s["work"] = torch.empty(case["batch"] * (case["dim"] + 16) + 256, dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty(case["batch"], case["codebooks"], case["vocab"], device="cuda")
        return s
    S, N, H, K, D, page = (case[n] for n in ("streams", "new", "heads", "kv_heads", "dim", "page"))
    low = 0 if S > 1 and N > 1 else 1   # a stream of a batch may be without new tokens
    many = torch.randint(low, N + 1, (S,), generator=g, device="cuda") if case["ragged"] else torch.full((S,), N, device="cuda")
    cached = torch.randint(case["least"], case["most"] + 1, (S,), generator=g, device="cuda")
    wide = -(-(case["most"] + N) // page)   # pages of the longest stream
    rows = S * N                            # rows behind the last stream's tokens stay as they are
    s["rows"], s["pages"] = rows, wide
    start = torch.zeros(S + 1, dtype=torch.int64, device="cuda")
    start[1:] = many.cumsum(0)
    s["start"], s["length"] = start.to(torch.int32), (cached + many).to(torch.int32)
    table = torch.randperm(S * wide, generator=g, device="cuda").view(S, wide).to(torch.int32)
    if case.get("window"):
        # pages that the window has left behind are given back
        last = torch.div((cached - case["window"] + 1).clamp(min=0), page, rounding_mode="floor")
        table[torch.arange(wide, device="cuda") < last[:, None]] = -1
    s["table"] = table
    s["k_pages"], s["v_pages"] = (torch.randn(S * wide, K, page, D, generator=g, device="cuda", dtype=t) for _ in range(2))

    def rows_of(width, extra):
        return normal(rows, width + extra).to(t)

    s["q"] = rows_of(H * D, case["pad"])[:, :H * D]
    if case["op"] == "append":
        kv = rows_of(2 * K * D, case["pad"])
        s["k"], s["v"] = kv[:, :K * D], kv[:, K * D:2 * K * D]
        s["q_out"] = torch.zeros(rows, H * D, dtype=t, device="cuda")
        s["freq"] = torch.tensor([THETA ** (-2 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=torch.float32, device="cuda")
        s["q_weight"], s["k_weight"] = (1 + 0.1 * normal(D) for _ in range(2))
    else:
        s["gate_values"] = normal(rows, H).to(t) if case["gate"] else None
        s["out"] = torch.zeros(rows, H * D, dtype=t, device="cuda")
    if own:
        Z = _library()
        s["cache"] = Z.PagedCache(s["k_pages"], s["v_pages"], s["table"], s["length"], s["start"])
    return s


def _tokens(s):
    """[streams, new]: each stream's rows (past its last: the row behind all), and their positions."""
    i = torch.arange(s["new"], device=s["start"].device)
    start, many = s["start"][:-1, None].long(), (s["start"][1:] - s["start"][:-1])[:, None].long()
    row = torch.where(i < many, start + i, s["rows"])
    return row, s["length"][:, None].long() - many + i


def _put(rows, where, values):
    """rows with values at the rows `where` (one past the end: nowhere)."""
    wide = torch.cat([rows, rows[:1]])
    wide[where.reshape(-1)] = values.reshape(-1, rows.shape[1])
    rows.copy_(wide[:-1])


def _take(rows, where):
    return rows[where.clamp(max=rows.shape[0] - 1)]


def _append(s):
    S, N, H, K, D, page, R = (s[n] for n in ("streams", "new", "heads", "kv_heads", "dim", "page", "rot"))
    row, at = _tokens(s)
    angle = at.double()[..., None] * s["freq"].double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    first = slice(0, R // 2) if s["halves"] else slice(0, R, 2)
    second = slice(R // 2, R) if s["halves"] else slice(1, R, 2)

    def turned(x, heads, weight):
        x = _take(x, row).float().view(S, N, heads, D)
        if s["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        a, b = x[..., first], x[..., second]
        y = x.clone()
        y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
        return y.to(_type(s))

    _put(s["q_out"], row, turned(s["q"], H, s["q_weight"]))
    live = row < s["rows"]
    slot = at.clamp(min=0)
    pages = s["table"].long().gather(1, torch.div(slot, page, rounding_mode="floor").clamp(max=s["pages"] - 1))
    # [pages * kv heads * page] rows of D
    where = (pages[..., None] * K + torch.arange(K, device=row.device)) * page + (slot % page)[..., None]
    total = s["k_pages"].shape[0] * K * page
    where = torch.where(live[..., None], where, total)
    _put(s["k_pages"].view(total, D), where, turned(s["k"], K, s["k_weight"]))
    _put(s["v_pages"].view(total, D), where, _take(s["v"], row).reshape(S, N, K, D))
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    S, N, H, K, D, page = (s[n] for n in ("streams", "new", "heads", "kv_heads", "dim", "page"))
    G, L = H // K, s["pages"] * page
    row, at = _tokens(s)
    table = s["table"].long().clamp(min=0)
    j = torch.arange(L, device=row.device)
    held = (s["table"] >= 0).repeat_interleave(page, 1) & (j < s["length"][:, None])           # [S, L]
    k = s["k_pages"][table].transpose(1, 2).reshape(S, K, L, D).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(S, K, L, D).float().masked_fill(~held[:, None, :, None], 0)
    q = _take(s["q"], row).float().view(S, N, K, G, D).permute(0, 2, 1, 3, 4).reshape(S, K, N * G, D)
    sees = held[:, None] & (j <= at[..., None])                                                 # [S, N, L]
    if s["window"]:
        sees = sees & (j > at[..., None] - s["window"])
    x = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(D)).view(S, K, N, G, L)
    x = x.masked_fill_(~sees[:, None, :, None], -math.inf)
    most = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = x.sum(-1, keepdim=True)
    y = (x.view(S, K, N * G, L) @ v).view(S, K, N, G, D) / torch.where(total == 0, 1.0, total)
    y = y.permute(0, 2, 1, 3, 4).reshape(S, N, H, D)
    if s["gate_values"] is not None:
        y = y / (1 + torch.exp(-_take(s["gate_values"], row).float()))[..., None]
    _put(s["out"], row, y.to(_type(s)))
    return s["out"]


def _head8(s):
    C, V = s["codebooks"], s["vocab"]
    x = s["hidden"].double()
    most = x.abs().amax(1, keepdim=True)
    # sums of 1024 products of 8-bit integers are exact in 32 bits
    q = torch.round(127 * x / torch.where(most == 0, 1.0, most)).float()
    W = s["W"].view(C, s["rows"], -1)[:, :V].reshape(C * V, -1).float()
    y = 0
    for at in range(0, s["dim"], 1024):
        y = y + (q[:, at:at + 1024] @ W[:, at:at + 1024].t()).double()
    y = (y * (most / 127).float()).float() * s["w_scale"].view(C, s["rows"])[:, :V].reshape(-1)
    return (CAP * torch.tanh(y / CAP)).view(-1, C, V)


def run(state):
    s = state
    if not own:
        return {"append": _append, "attend": _attend, "head8": _head8}[s["op"]](s)
    Z = _library()
    if s["op"] == "append":
        Z.cache_append(s["cache"], s["q"], s["k"], s["v"], s["q_out"], freq=s["freq"], halves=s["halves"],
                       q_weight=s["q_weight"] if s["norm"] else None, k_weight=s["k_weight"] if s["norm"] else None,
                       eps=EPS if s["norm"] else -1.0)
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["op"] == "attend":
        Z.cache_attend(s["cache"], s["q"], s["out"], window=s["window"], gate=s["gate_values"], max_new=s["new"])
        return s["out"]
    Z.head_i8(s["W"], s["w_scale"], s["rows"], s["codebooks"], s["vocab"], s["hidden"], s["out"], s["work"])
    return s["out"]


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "head8":
        b, d, n = case["batch"], case["dim"], case["codebooks"] * case["vocab"]
        return {"bytes": n * (d + 4) + size * b * d + 4 * b * n, "flops": 2 * b * n * d}
    S, H, K, D = (case[n] for n in ("streams", "heads", "kv_heads", "dim"))
    least_new = (0 if S > 1 and case["new"] > 1 else 1) if case["ragged"] else case["new"]
    new, cached = (least_new + case["new"]) / 2, (case["least"] + case["most"]) / 2
    if case["op"] == "append":
        return {"bytes": 2 * size * S * new * (H + 2 * K) * D, "flops": S * new * (H + K) * D * 10}
    # keys that a chunk's rows see, and how many of them one row does on average
    seen, each = cached + new, cached + (new + 1) / 2
    if case["window"]:
        each = min(each, case["window"])
        seen = min(seen, case["window"] + new)
    gate = S * new * H if case["gate"] else 0
    return {"bytes": size * (2 * S * new * H * D + gate + 2 * S * seen * K * D), "flops": 4 * S * new * each * H * D}


def _exact_stream(s, i):
    """(the stream's rows, its tokens' positions)."""
    a, b, n = int(s["start"][i]), int(s["start"][i + 1]), int(s["length"][i])
    return slice(a, b), torch.arange(n - (b - a), n, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "head8":
        h = s["hidden"].double()
        scale = h.abs().max(dim=1).values / 127
        whole = torch.special.round(h / torch.where(scale > 0, scale, 1.0)[:, None])
        # a quotient that 64 bits put next to a half is settled by whole numbers of its own: 254 x against an odd multiple of the largest
        odd = 2 * torch.floor(h / torch.where(scale > 0, scale, 1.0)[:, None]) + 1
        tie = (254 * h == odd * h.abs().max(dim=1).values[:, None]) & (scale > 0)[:, None]
        low = (odd - 1) / 2
        whole = torch.where(tie, torch.where(low % 2 == 0, low, low + 1), whole)
        keep = torch.cat([torch.arange(c * case["rows"], c * case["rows"] + case["vocab"], device="cuda") for c in range(case["codebooks"])])
        y = torch.mm(whole, s["W"][keep].double().t()) * scale[:, None] * s["w_scale"][keep].double()
        return (CAP * torch.tanh(y / CAP)).view(-1, case["codebooks"], case["vocab"])
    H, K, D, page = (case[n] for n in ("heads", "kv_heads", "dim", "page"))
    if case["op"] == "append":
        q_out, k_pages, v_pages = s["q_out"].double(), s["k_pages"].double(), s["v_pages"].double()
        for i in range(case["streams"]):
            rows, at = _exact_stream(s, i)
            turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), at[:, None].double() * s["freq"].double())[:, None]

            def rotated(x, weight):
                x = x.double()
                if case["norm"]:
                    x = x * (x.pow(2).sum(-1, keepdim=True) / D + float(np.float32(EPS))).rsqrt() * weight.double()
                r = x[..., :case["rot"]]
                pairs = torch.complex(*(r.chunk(2, -1) if case["halves"] else r.unflatten(-1, (-1, 2)).unbind(-1))) * turn
                r = torch.cat([pairs.real, pairs.imag], -1) if case["halves"] else torch.view_as_real(pairs).flatten(-2)
                return torch.cat([r, x[..., case["rot"]:]], -1)

            many = at.numel()
            q_out[rows] = rotated(s["q"][rows].reshape(many, H, D), s["q_weight"]).flatten(1)
            pages = s["table"][i].long()[torch.div(at, page, rounding_mode="floor")]
            k_pages[pages, :, at % page] = rotated(s["k"][rows].reshape(many, K, D), s["k_weight"])
            v_pages[pages, :, at % page] = s["v"][rows].reshape(many, K, D).double()
        return {"q": q_out, "k_pages": k_pages, "v_pages": v_pages}
    out = s["out"].double()
    for i in range(case["streams"]):
        rows, at = _exact_stream(s, i)
        many, length = at.numel(), int(s["length"][i])
        if many == 0:
            continue
        first = max(0, int(at[0]) - case["window"] + 1) if case["window"] else 0
        j = torch.arange(first, length, device="cuda")
        pages = s["table"][i].long()[torch.div(j, page, rounding_mode="floor")]
        k, v = (s[n][pages, :, j % page].double() for n in ("k_pages", "v_pages"))             # [keys, K, D]
        hidden = j[None] > at[:, None]
        if case["window"]:
            hidden = hidden | (j[None] + case["window"] <= at[:, None])
        for h in range(H):
            x = torch.mm(s["q"][rows, h * D:(h + 1) * D].double(), k[:, h // (H // K)].t()) / D ** 0.5
            y = torch.mm(torch.softmax(x.masked_fill(hidden, -math.inf), dim=1), v[:, h // (H // K)])
            if case["gate"]:
                y = y * torch.sigmoid(s["gate_values"][rows, h:h + 1].double())
            out[rows, h * D:(h + 1) * D] = y
    return out
