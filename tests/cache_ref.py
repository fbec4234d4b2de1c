"""The paged cache's calls evaluated in 64 bits from their definitions, on the CPU, with bounds of what f32
arithmetic and the stated roundings can add."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}   # half a step, relative


class Cache:
    """Host copies of a paged cache's tensors."""

    def __init__(self, k, v, table, kv_len, q_start):
        self.k, self.v = k.cpu(), v.cpu()
        self.table, self.kv_len, self.q_start = (t.cpu().long().numpy() for t in (table, kv_len, q_start))
        self.pages, self.heads, self.page, self.dim = self.k.shape

    def streams(self, rows):
        """(stream, first row, rows, tokens) of each stream with new tokens."""
        for s in range(len(self.kv_len)):
            a, b = int(self.q_start[s]), int(self.q_start[s + 1])
            assert 0 <= a <= b <= rows
            if b > a:
                yield s, a, b - a, max(0, int(self.kv_len[s]))

    def place(self, s, j):
        """(page, slot) of a stream's token, or None."""
        if j < 0 or j >= self.table.shape[1] * self.page:
            return None
        p = int(self.table[s, j // self.page])
        return (p, j % self.page) if 0 <= p < self.pages else None


def rotated(x, pos, weight, eps, freq, halves):
    """(y, bound) of one head's rows x [n, dim] at positions pos [n]: y and what f32 may be off."""
    x = x.double()
    if eps >= 0:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + float(np.float32(eps)))
        if weight is not None:
            x = x * weight.double()
    y, size = x.clone(), x.abs()
    if freq is not None and freq.numel():
        n = freq.numel()
        t = pos.double()[:, None] * freq.double()
        first = torch.arange(n) if halves else 2 * torch.arange(n)
        second = first + n if halves else first + 1
        a, b = x[:, first], x[:, second]
        y[:, first] = a * torch.cos(t) - b * torch.sin(t)
        y[:, second] = b * torch.cos(t) + a * torch.sin(t)
        size[:, first] = size[:, second] = a.abs() + b.abs()
    # a norm of a few f32 roundings and sums of up to 256 squares in a tree, sines to 2^-22: 2^-19 in all
    return y, size * 2.0 ** -19


def append(c, rows, q, k, v, q_weight, k_weight, eps, freq, halves):
    """(q, its bound, keys, their bounds, values): what the call leaves, starting from zeros for q
    and the cache's own pages."""
    t = c.k.dtype
    q_out, q_tol = torch.zeros(rows, 0 if q is None else q.shape[1], dtype=torch.float64), None
    q_tol = torch.zeros_like(q_out)
    keys, values = c.k.double().clone(), c.v.clone()
    k_tol = torch.zeros_like(keys)
    for s, a, n, length in c.streams(rows):
        pos = torch.arange(length - n, length)
        if q is not None:
            for h in range(q.shape[1] // c.dim):
                at = slice(h * c.dim, (h + 1) * c.dim)
                y, e = rotated(q[a:a + n, at], pos, q_weight, eps, freq, halves)
                q_out[a:a + n, at], q_tol[a:a + n, at] = y, e + HALF[t] * (y.abs() + e)
        for h in range(c.heads):
            at = slice(h * c.dim, (h + 1) * c.dim)
            y, e = rotated(k[a:a + n, at], pos, k_weight, eps, freq, halves)
            for i in range(n):
                where = c.place(s, int(pos[i]))
                if where is not None:
                    keys[where[0], h, where[1]] = y[i]
                    k_tol[where[0], h, where[1]] = e[i] + HALF[t] * (y[i].abs() + e[i])
                    values[where[0], h, where[1]] = v[a + i, at]
    return q_out, q_tol, keys, k_tol, values


def attend(c, rows, q, out, scale=None, window=0, gate=None):
    """(out, bound): the rows that the call writes in 64 bits, the others as they were."""
    t = c.k.dtype
    scale = c.dim ** -0.5 if scale is None else float(np.float32(scale))
    y, tol = out.cpu().double().clone(), torch.zeros(out.shape, dtype=torch.float64)
    heads = q.shape[1] // c.dim
    group = heads // c.heads
    for s, a, n, length in c.streams(rows):
        room = min(length, c.table.shape[1] * c.page)
        held = np.array([c.place(s, j) is not None for j in range(room)], bool)
        at = np.flatnonzero(held)
        where = [c.place(s, int(j)) for j in at]
        pages = torch.tensor([w[0] for w in where], dtype=torch.long)
        slots = torch.tensor([w[1] for w in where], dtype=torch.long)
        pos = torch.arange(length - n, length)
        j = torch.from_numpy(at)
        sees = j[None] <= pos[:, None]
        if window > 0:
            sees = sees & (j[None] > pos[:, None] - window)
        for h in range(heads):
            cols = slice(h * c.dim, (h + 1) * c.dim)
            k, v = c.k[pages, h // group, slots].double(), c.v[pages, h // group, slots].double()
            qr = q[a:a + n, cols].double()
            g = torch.ones(n, dtype=torch.float64)
            if gate is not None:
                g = 1 / (1 + torch.exp(-gate[a:a + n, h].double()))
            for i in range(n):
                on = sees[i]
                if not bool(on.any()):
                    y[a + i, cols] = 0
                    continue
                x = (k[on] @ qr[i]) * scale
                p = torch.softmax(x, 0)
                # what f32 may be off in a score: 2^-16 of its terms' sizes covers 256 of them added
                # one by one, and three-part products; in a weight twice that, and 2^-18 for its
                # exponential; a bf16 weight is rounded; the weights' and values' sums: 2^-24 a term
                off = 2 * 2.0 ** -16 * float(((k[on].abs() @ qr[i].abs()) * scale).max()) + 2.0 ** -18
                off = 2 * math.expm1(off) + (HALF[t] if t == torch.bfloat16 else 0.0) + 2.0 ** -24 * int(on.sum()) + 2.0 ** -18
                size = p @ v[on].abs()
                y[a + i, cols] = g[i] * (p @ v[on])
                e = g[i] * size * off
                tol[a + i, cols] = e + HALF[t] * (y[a + i, cols].abs() + e)
    return y, tol


def attend_whole(c, rows, q, out, scale=None, window=0, gate=None):
    """attend() by one product for all rows of a stream and query head: for many rows."""
    t = c.k.dtype
    scale = c.dim ** -0.5 if scale is None else float(np.float32(scale))
    y, tol = out.cpu().double().clone(), torch.zeros(out.shape, dtype=torch.float64)
    heads = q.shape[1] // c.dim
    group = heads // c.heads
    for s, a, n, length in c.streams(rows):
        room = min(length, c.table.shape[1] * c.page)
        at = [j for j in range(room) if c.place(s, j) is not None]
        if not at:
            y[a:a + n, :heads * c.dim] = 0
            continue
        where = torch.tensor([c.place(s, j) for j in at], dtype=torch.long)
        j, pos = torch.tensor(at), torch.arange(length - n, length)[:, None]
        sees = (j <= pos) & (j > pos - window) if window > 0 else j <= pos
        some = sees.any(1, keepdim=True)
        for h in range(heads):
            cols = slice(h * c.dim, (h + 1) * c.dim)
            k, v = (x[where[:, 0], h // group, where[:, 1]].double() for x in (c.k, c.v))
            qr = q[a:a + n, cols].double()
            x = (qr @ k.t() * scale).masked_fill(~sees, -math.inf)
            p = torch.softmax(torch.where(some, x, 0.0), 1) * sees
            g = 1.0 if gate is None else 1 / (1 + torch.exp(-gate[a:a + n, h:h + 1].double()))
            terms = ((qr.abs() @ k.abs().t()) * scale * sees).amax(1, keepdim=True)
            off = 2 * torch.expm1(2 * 2.0 ** -16 * terms + 2.0 ** -18) + (HALF[t] if t == torch.bfloat16 else 0.0)
            off = off + 2.0 ** -24 * sees.sum(1, keepdim=True) + 2.0 ** -18
            y[a:a + n, cols] = g * (p @ v)
            e = g * (p @ v.abs()) * off
            tol[a:a + n, cols] = e + HALF[t] * (y[a:a + n, cols].abs() + e)
    return y, tol
