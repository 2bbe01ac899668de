"""The paged 8-bit cache and the sampler in 64 bits on the CPU, token by token as they are defined (tests only)."""
import math

import numpy as np


def plan(lengths, new, block, table, free, count, capacity):
    """(context, query_start, table, positions, slots, count, status)."""
    table = table.copy()
    requests, width = table.shape
    status = 0
    if any(c < 0 or n < 0 for c, n in zip(lengths, new)):
        status = 3
    elif any(c + n > width * block for c, n in zip(lengths, new)):
        status = 2
    elif not 0 <= count <= len(free) or sum(new) > capacity:
        status = 3
    elif sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(lengths, new)) > count:
        status = 1
    if status:
        return list(lengths), [0] * (requests + 1), table, [0] * capacity, [-1] * capacity, count, status
    start, positions, slots = [0], [], []
    for r, (c, n) in enumerate(zip(lengths, new)):
        for pos in range(c, c + n):
            if pos % block == 0:
                count -= 1
                table[r, pos // block] = free[count]
            positions.append(pos)
            slots.append(int(table[r, pos // block]) * block + pos % block)
        start.append(len(slots))
    more = capacity - len(slots)
    return [c + n for c, n in zip(lengths, new)], start, table, positions + [0] * more, slots + [-1] * more, count, 0


def rotate(x, positions, freqs):
    """x [tokens, heads, dim] float64: entries d and d + n turn by position * freq."""
    n = len(freqs)
    angle = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float32).astype(np.float64)
    y = x.copy()
    y[..., :n] = x[..., :n] * np.cos(angle) - x[..., n:2 * n] * np.sin(angle)
    y[..., n:2 * n] = x[..., :n] * np.sin(angle) + x[..., n:2 * n] * np.cos(angle)
    return y


class Store:
    """One side (keys or values) of a cache: codes [page, token, head, dim], scales [page, head] f32."""

    def __init__(self, pages, block, heads, dim):
        self.block = block
        self.codes = np.zeros((pages, block, heads, dim), np.float64)
        self.scales = np.zeros((pages, heads), np.float32)

    def append(self, x, slots):
        """x [tokens, heads, dim] float64.  A stretch of ascending slots in a page is stored at once."""
        t = 0
        while t < len(slots):
            if not 0 <= slots[t] < self.codes.shape[0] * self.block:
                t += 1
                continue
            n = 1
            page, at = divmod(slots[t], self.block)
            while t + n < len(slots) and slots[t + n] == slots[t] + n and at + n < self.block:
                n += 1
            v = np.where(np.isnan(x[t:t + n]), 0.0, x[t:t + n])
            largest = np.where(np.isfinite(v), np.abs(v), 0.0).max((0, 2))
            before = np.zeros_like(self.scales[page]) if at == 0 else self.scales[page]
            scale = np.maximum(before, (largest / 127.0).astype(np.float32))
            with np.errstate(divide="ignore", invalid="ignore"):
                for h in range(v.shape[1]):
                    s, b = float(scale[h]), float(before[h])
                    if s > b and at > 0:
                        self.codes[page, :at, h] = np.rint(self.codes[page, :at, h] * b / s)
                    self.codes[page, at:at + n, h] = np.clip(np.rint(v[:, h] / s), -127, 127) if s > 0 else 0.0
            self.scales[page] = scale
            t += n

    def rows(self, slots):
        page, at = np.divmod(np.asarray(slots), self.block)
        return (self.codes[page, at].astype(np.float32) * self.scales[page][..., None]).astype(np.float32)


def key_layout(codes):
    """[page, token, head, dim] -> int8 [page, head, dim / 16, token, 16]."""
    p, b, h, d = codes.shape
    return np.ascontiguousarray(codes.reshape(p, b, h, d // 16, 16).transpose(0, 2, 3, 1, 4)).astype(np.int8)


def value_layout(codes):
    """[page, token, head, dim] -> int8 [page, head, token / 16, dim, 16]."""
    p, b, h, d = codes.shape
    return np.ascontiguousarray(codes.reshape(p, b // 16, 16, h, d).transpose(0, 3, 1, 4, 2)).astype(np.int8)


def attention(q, start, context, table, block, k, v, scale, window, out):
    """q [tokens, heads, dim] float64; k, v [page, token, kv head, dim] float64 values; out [tokens, heads, dim] float64, updated."""
    group = q.shape[1] // k.shape[2]
    pages = k.shape[0]
    for r, c in enumerate(context):
        rows = start[r + 1] - start[r]
        if rows == 0:
            continue
        c = max(c, 0)
        at = np.arange(c)
        page = table[r, at // block] if c else np.zeros(0, np.int64)
        there = (page >= 0) & (page < pages)
        kk, vv = k[np.where(there, page, 0), at % block], v[np.where(there, page, 0), at % block]
        for i in range(rows):
            pos = context[r] - rows + i
            seen = there & (at <= pos) & ((at > pos - window) if window else True)
            for h in range(q.shape[1]):
                if not seen.any():
                    out[start[r] + i, h] = 0.0
                    continue
                z = (kk[seen, h // group] @ q[start[r] + i, h]) * scale
                w = np.exp(z - z.max())
                out[start[r] + i, h] = (w @ vv[seen, h // group]) / w.sum()
    return out


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, float64 of its f32 or bf16 values: (token, log-probability, gap to the nearest border of the choice in weight)."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    top = x.max()
    if top == -np.inf:
        return -1, -math.inf, 1.0
    if not temperature > np.finfo(np.float32).eps:
        return int(np.argmax(x)), 0.0, 1.0
    order = np.argsort(-x, kind="stable")
    with np.errstate(invalid="ignore"):
        e = np.where(x[order] == top, 0.0, (x[order] - top) / temperature)
    w = np.where(x[order] > -np.inf, np.exp(e), 0.0)
    gap = 1.0
    n = min(top_k, len(w)) if top_k > 0 else len(w)
    if top_p < 1:
        sums = np.cumsum(w[:n])
        want = max(top_p, 0.0) * sums[-1]
        gap = min(gap, float(np.min(np.abs(sums - want)) / sums[-1])) if top_p > 0 else gap
        n = min(int(np.searchsorted(sums, want)) + 1, n)
    if min_p > 0:
        border = min(min_p, 1.0)
        n = min(n, int((w[:n] >= border).sum()))
    sums = np.cumsum(w[:n])
    want = min(max(u, 0.0), 1.0) * sums[-1]
    if 0 < u < 1:
        gap = min(gap, float(np.min(np.abs(sums - want)) / sums[-1]))
    at = min(int(np.searchsorted(sums, want, side="right")), n - 1)
    while w[at] == 0.0 and at > 0:
        at -= 1
    return int(order[at]), float(np.log(w[at] / sums[-1])), gap
