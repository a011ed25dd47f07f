"""The row operators from their definitions, one row at a time in 64 bits (test infrastructure only)."""
import numpy as np


def sort(ids, first, experts, align, rows):
    """counts, offsets, position, source of a [tokens, choices] array of expert numbers."""
    ids = np.asarray(ids)
    flat = [int(e) for e in ids.reshape(-1)]
    held = [[] for _ in range(experts)]
    for a, e in enumerate(flat):
        if first <= e < first + experts:
            held[e - first].append(a)
    counts = np.array([len(h) for h in held], dtype=np.int32)
    offsets = np.zeros(experts + 1, dtype=np.int32)
    position = np.full(len(flat), -1, dtype=np.int32)
    source = np.full(rows, -1, dtype=np.int32)
    for e, h in enumerate(held):
        offsets[e + 1] = offsets[e] + (len(h) + align - 1) // align * align
        for i, a in enumerate(h):
            r = offsets[e] + i
            if r < rows:
                position[a] = r
                source[r] = a
    return counts, offsets, position.reshape(ids.shape), source


def dispatch(x, position, source, y):
    """y after the rows of x have moved."""
    y = y.copy()
    y[source < 0] = 0
    for t in range(position.shape[0]):
        for p in position[t]:
            if 0 <= p < y.shape[0]:
                y[p] = x[t]
    return y


def combine(y, position, weights=None):
    """(sum, sum of the terms' sizes) for every token, in 64 bits."""
    out = np.zeros((position.shape[0], y.shape[1]))
    size = np.zeros_like(out)
    for t in range(position.shape[0]):
        for k, p in enumerate(position[t]):
            if 0 <= p < y.shape[0]:
                term = y[p].astype(np.float64) * (1.0 if weights is None else np.float64(weights[t, k]))
                out[t] += term
                size[t] += np.abs(term)
    return out, size


def combine_backward(y, dout, position, source, weights, dy):
    """(dy, dweights, sum of the sizes of dweights' terms) in 64 bits; dy starts as what the buffer held."""
    dy = dy.astype(np.float64)
    dy[source < 0] = 0
    dw = np.zeros(position.shape)
    size = np.zeros(position.shape)
    for t in range(position.shape[0]):
        for k, p in enumerate(position[t]):
            if 0 <= p < dy.shape[0]:
                g = dout[t].astype(np.float64)
                dy[p] = g * np.float64(weights[t, k])
                dw[t, k] = (g * y[p]).sum()
                size[t, k] = np.abs(g * y[p]).sum()
    return dy, dw, size


def tables(cached, added, page, free, tables, tokens):
    """(tables, starts, used, slots, positions) after the new tokens have their pages."""
    tables = tables.copy()
    most = 2 ** 31 - 1
    starts, taken, flat = [0], 0, []
    for b in range(len(cached)):
        c, n = max(int(cached[b]), 0), max(int(added[b]), 0)
        owned, want = (min(-(-x // page), tables.shape[1]) for x in (c, min(c + n, most)))
        for j in range(owned, want):
            at = taken + j - owned
            tables[b, j] = free[at] if at < len(free) else -1
        taken = min(taken + want - owned, most)
        starts.append(min(starts[-1] + n, most))
        for p in range(c, c + min(n, tokens)):
            p = min(p, most)
            j = p // page
            at = int(tables[b, j]) if j < tables.shape[1] else -1
            flat.append((at * page + p % page if at >= 0 else -1, p))
    flat = (flat + [(-1, -1)] * tokens)[:tokens]
    return (tables, np.array(starts, dtype=np.int32), np.array([taken], dtype=np.int32),
            np.array([s for s, _ in flat], dtype=np.int64), np.array([p for _, p in flat], dtype=np.int32))


def store(cache, slots, rows):
    """cache [pages, page, heads, width] after rows [tokens, heads, width] have gone to their slots."""
    cache = cache.copy()
    flat = cache.reshape((-1,) + cache.shape[2:])
    for t, s in enumerate(slots):
        if 0 <= s < flat.shape[0]:
            flat[s] = rows[t]
    return cache


def load(cache, slots):
    flat = cache.reshape((-1,) + cache.shape[2:])
    rows = np.zeros((len(slots),) + cache.shape[2:], dtype=cache.dtype)
    for t, s in enumerate(slots):
        if 0 <= s < flat.shape[0]:
            rows[t] = flat[s]
    return rows
