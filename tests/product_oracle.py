"""The products from their definitions, in 64 bits (test infrastructure only)."""
import numpy as np


def bounds(offsets, rows):
    """First and last-plus-one row of every group."""
    o = np.clip(np.asarray(offsets, dtype=np.int64), 0, rows)
    return [(int(a), max(int(a), int(b))) for a, b in zip(o[:-1], o[1:])]


def grouped(x, w, offsets, transposed, y):
    """(y after the product, sum of the terms' sizes); rows of no group keep what y held."""
    y, size = np.array(y, dtype=np.float64), np.zeros(y.shape)
    x, w = np.asarray(x, dtype=np.float64), np.asarray(w, dtype=np.float64)
    for e, (lo, hi) in enumerate(bounds(offsets, x.shape[0])):
        m = w[e].T if transposed else w[e]
        if lo < hi:
            y[lo:hi] = x[lo:hi] @ m
            size[lo:hi] = np.abs(x[lo:hi]) @ np.abs(m)
    return y, size


def weights(x, dy, offsets, groups):
    """(dw, sum of the terms' sizes)"""
    x, dy = np.asarray(x, dtype=np.float64), np.asarray(dy, dtype=np.float64)
    dw = np.zeros((groups, x.shape[1], dy.shape[1]))
    size = np.zeros_like(dw)
    for e, (lo, hi) in enumerate(bounds(offsets, x.shape[0])):
        if lo < hi:
            dw[e] = x[lo:hi].T @ dy[lo:hi]
            size[e] = np.abs(x[lo:hi]).T @ np.abs(dy[lo:hi])
    return dw, size


def seen(position, owner, table, pages, page, window):
    """The (page, slot) pairs that a query sees."""
    if position < 0 or not 0 <= owner < table.shape[0]:
        return []
    first = max(0, position - window + 1) if window else 0
    at = [(int(table[owner, t // page]), t % page) for t in range(first, min(position + 1, table.shape[1] * page))]
    return [(p, s) for p, s in at if 0 <= p < pages]


def attend(q, k, v, table, owners, positions, window, scale):
    """q [queries, heads, width], k and v [pages, page, key heads, width] -> out, log sums, and what an error of the scores or of a sum can come to:
    the weighted sum of the values' sizes, the largest size of a score's terms, the tokens seen and the largest value."""
    queries, heads, width = q.shape
    pages, page, key_heads = k.shape[:3]
    out = np.zeros(q.shape)
    logs = np.full((queries, heads), -np.inf)
    size, terms, count, most = np.zeros(q.shape), np.zeros((queries, heads)), np.zeros(queries, dtype=np.int64), np.zeros(q.shape)
    for i in range(queries):
        at = seen(int(positions[i]), int(owners[i]), table, pages, page, window)
        count[i] = len(at)
        if not at:
            continue
        p, s = np.array(at).T
        for h in range(heads):
            kh = k[p, s, h // (heads // key_heads)].astype(np.float64)
            vh = v[p, s, h // (heads // key_heads)].astype(np.float64)
            query = q[i, h].astype(np.float64)
            score = scale * (kh @ query)
            top = score.max()
            logs[i, h] = top + np.log(np.exp(score - top).sum())
            weight = np.exp(score - logs[i, h])
            out[i, h] = weight @ vh
            size[i, h] = weight @ np.abs(vh)
            most[i, h] = np.abs(vh).max(axis=0)
            terms[i, h] = abs(scale) * (np.abs(kh) @ np.abs(query)).max()
    return out, logs, size, terms, count, most
