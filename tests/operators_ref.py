"""Plain 64-bit restatements of the head with adapters, the block-tail norm and the draft
verification, from their formulas; numpy on the host."""
import numpy as np


def head_adapters(W, rows_per_cb, n_cb, vocab, h, A, B, ids, scale, softcap):
    """Logits [batch, n_cb, vocab], and the sums of the absolute terms of the two products."""
    W = W.astype(np.float64).reshape(n_cb, rows_per_cb, -1)[:, :vocab].reshape(n_cb * vocab, -1)
    A, h = A.astype(np.float64), h.astype(np.float64)
    B = B.astype(np.float64).reshape(len(A), n_cb, rows_per_cb, -1)[:, :, :vocab]
    B = B.reshape(len(A), n_cb * vocab, -1)
    y, mag, low = h @ W.T, np.abs(h) @ np.abs(W).T, np.zeros((len(h), n_cb * vocab))
    for b, a in enumerate(ids):
        if 0 <= a < len(A):
            f = 1.0 if scale is None else float(scale[a])
            y[b] += f * (B[a] @ (A[a] @ h[b]))
            low[b] = abs(f) * (np.abs(B[a]) @ (np.abs(A[a]) @ np.abs(h[b])))
    lg = softcap * np.tanh(y / softcap) if softcap > 0 else y
    shape = (len(h), n_cb, vocab)
    return lg.reshape(shape), mag.reshape(shape), low.reshape(shape)


def block_norm(resid, block, post_weight, post_eps, gate, sigmoid, scale, norm_weight, norm_eps):
    """r, n and the magnitude of r's second term, [rows, dim] f64."""
    x, y = resid.astype(np.float64), block.astype(np.float64)
    if post_eps >= 0:
        y = y / np.sqrt((y * y).mean(1, keepdims=True) + np.float64(np.float32(post_eps)))
        if post_weight is not None:
            y = y * post_weight.astype(np.float64)
    if gate is not None:
        g = np.broadcast_to(gate, x.shape).astype(np.float64)
        y = y * (1 / (1 + np.exp(-g)) if sigmoid else g)
    y = y * np.float64(np.float32(scale))
    r = x + y
    n = r / np.sqrt((r * r).mean(1, keepdims=True) + np.float64(np.float32(norm_eps)))
    if norm_weight is not None:
        n = n * norm_weight.astype(np.float64)
    return r, n, np.abs(y)


def _distribution(lg, seen, may, p):
    """The sampler's list of one row: tokens in order, their kept weights (unnormalised), flag."""
    f32, x = np.float32, lg.astype(np.float32).copy()
    odd = ~(x < np.inf)
    x[odd] = -np.inf
    rho = f32(p.repetition_penalty)
    if rho != 1:
        with np.errstate(over="ignore"):
            pen = np.where(x > 0, x * (f32(1) / rho), x * rho).astype(np.float32)
        x = np.where(seen, np.minimum(pen, f32(3.4028235e38)), x)
    x = np.where(may, x, -np.inf).astype(np.float32)
    flag, top = 2 * int(odd.any()), x.max()
    if not top >= -1e9:
        return np.array([p.pad_id]), np.array([1.0]), flag | 1
    order = np.lexsort((np.arange(len(x)), -x.astype(np.float64)))
    order = order[: int((x > -np.inf).sum())]
    if p.top_k > 0:
        order = order[: p.top_k]
    e = np.exp((x[order].astype(np.float64) - np.float64(top)) * (1.0 / np.float64(f32(p.temperature))))
    keep = e >= np.float64(f32(p.min_p))
    if p.top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(e)[:-1]])
        inside = before < np.float64(f32(p.top_p)) * e.sum()
        inside[0] = True
        keep &= inside
    return order[keep], e[keep], flag


def verify_drafts(logits, vocab, p, drafts, u, probs=None, n_drafts=None, hist=None, hist_pos=None,
                  allow=None, delay_step=-1):
    """codes, accepted, flags, hist, hist_pos after the call."""
    S, D1, C, _ = logits.shape
    D = D1 - 1
    codes, flags = np.full((S, D1, C), -1, np.int32), np.zeros((S, D1, C), np.int32)
    accepted = np.zeros(S, np.int32)
    hist = None if hist is None else hist.copy()
    hist_pos = None if hist_pos is None else hist_pos.copy()
    H = 0 if hist is None else hist.shape[-1]
    for s in range(S):
        have = D if n_drafts is None else int(np.clip(n_drafts[s], 0, D))
        bits = np.ones(vocab, bool)
        if allow is not None:
            bits = (allow[s].view(np.uint32)[np.arange(vocab) >> 5] >> (np.arange(vocab) & 31).astype(np.uint32)) & 1 > 0
        pos = int(hist_pos[s]) % H if H else 0
        for d in range(have + 1):
            whole = d < have
            for c in range(C):
                seen = np.zeros(vocab, bool)
                if H:
                    row = hist[s, c].copy()
                    for j in range(d):
                        row[(pos + j) % H] = drafts[s, j, c]
                    seen[row[(row >= 0) & (row < vocab)]] = True
                may = bits
                if delay_step >= 0 and delay_step + d < c:
                    may = bits & (np.arange(vocab) == p.pad_id)
                tok, w, flag = _distribution(logits[s, d, c, :vocab], seen, may, p)
                flags[s, d, c] = flag
                total = w.sum()
                t = int(drafts[s, d, c]) if d < have else -1
                if d < have and 0 <= t < vocab:
                    q = 1.0 if probs is None else float(probs[s, d, c, t])
                    if np.float64(u[s, d, c, 0]) * q * total < w[tok == t].sum():
                        codes[s, d, c] = t
                        continue
                whole = False
                if d < have and not flag & 1:
                    q = (tok == t).astype(np.float64) if probs is None else probs[s, d, c, tok].astype(np.float64)
                    left = w - q * total
                    left = np.where(left > 0, left, 0.0)
                    if left.sum() > 0:
                        w = left
                at = np.flatnonzero((np.cumsum(w) >= np.float64(u[s, d, c, 1]) * w.sum()) & (w > 0))
                codes[s, d, c] = tok[at[0]] if len(at) else tok[np.flatnonzero(w > 0)[-1]]
            if not whole:
                break
        accepted[s] = d
        if H:
            for k in range(d + 1):
                hist[s, :, (pos + k) % H] = codes[s, k]
            hist_pos[s] = (pos + d + 1) % H
    return codes, accepted, flags, hist, hist_pos
