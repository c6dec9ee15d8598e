"""Decoding along branches in plain Python and numpy, in 64 bits: what the kernels of ``garuda_b200/kernels/branches.py`` are checked against."""
import math

import numpy as np


def layout(parents, cu_q, kv_lens, window=0):
    """(positions [T], reads: a list of sets of token numbers) of a step's trees."""
    positions, reads = [], []
    for r in range(len(kv_lens)):
        q_len = cu_q[r + 1] - cu_q[r]
        ctx = kv_lens[r] - q_len
        for i in range(q_len):
            chain, at = [], i
            while at is not None and at >= 0:
                chain.append(at)
                above = parents[cu_q[r] + at]
                at = above if above == -1 or 0 <= above < at else None
            rooted = at == -1
            positions.append(ctx + (len(chain) - 1 if rooted else 0))
            reads.append(set(chain[:window] if window else chain) if rooted else set())
    return positions, reads


def mask_words(reads, words):
    out = np.zeros((len(reads), words), dtype=np.uint32)
    for t, seen in enumerate(reads):
        for j in seen:
            out[t, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def attention(q, k_pool, v_pool, table, cu_q, kv_lens, positions, reads, scale, window=0):
    """``out [T, Hq, hd]`` in 64 bits, and what bounds its errors: ``sum_j p_j |v_j|`` of the same shape and, per (token, head), the largest
    ``scale sum_c |q_c k_c|`` of the keys that it reads. Pages that are not there (outside the pool) are zeros."""
    T, heads, hd = q.shape
    pages, kv_heads, page, _ = k_pool.shape
    group = heads // kv_heads
    out, weight, size = np.zeros((T, heads, hd)), np.zeros((T, heads, hd)), np.zeros((T, heads))
    for r in range(len(kv_lens)):
        n, a, b = int(kv_lens[r]), int(cu_q[r]), int(cu_q[r + 1])
        ctx = n - (b - a)
        where = [int(table[r, p // page]) if p // page < table.shape[1] else -1 for p in range(n)]
        k, v = np.zeros((n, kv_heads, hd)), np.zeros((n, kv_heads, hd))
        for p, at in enumerate(where):
            if 0 <= at < pages:
                k[p], v[p] = k_pool[at, :, p % page], v_pool[at, :, p % page]
        for t in range(a, b):
            first = max(0, positions[t] + 1 - window) if window else 0
            keys = list(range(min(first, ctx), ctx)) + sorted(ctx + j for j in reads[t] if ctx + j < n)
            if not keys:
                continue
            kk, vv = k[keys], v[keys]
            for h in range(heads):
                with np.errstate(invalid="ignore"):
                    s = scale * (kk[:, h // group] @ q[t, h])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t, h] = w @ vv[:, h // group]
                    weight[t, h] = w @ np.abs(vv[:, h // group])
                    size[t, h] = scale * (np.abs(kk[:, h // group]) @ np.abs(q[t, h])).max()
    return out, weight, size


def accept(tokens, targets, parents, cu_q):
    """(paths: a list per request, the tokens that come next)."""
    paths, after = [], []
    for r in range(len(cu_q) - 1):
        a, q_len = cu_q[r], cu_q[r + 1] - cu_q[r]
        path = [0] if q_len else []
        while path:
            more = [i for i in range(path[-1] + 1, q_len) if parents[a + i] == path[-1] and tokens[a + i] == targets[a + path[-1]]]
            if not more:
                break
            path.append(more[0])
        paths.append(path)
        after.append(targets[a + path[-1]] if path else -1)
    return paths, after


def move_rows(pool, table, page, ctx, path):
    """Rows ctx + path[i] of ``pool [calls, pages, heads, page, width]`` to ctx + i, all read before any is written."""
    pages = pool.shape[1]

    def place(slot):
        at = int(table[slot // page]) if slot // page < len(table) else -1
        return (at, slot % page) if 0 <= at < pages else None

    rows = [None if place(ctx + p) is None else pool[:, place(ctx + p)[0], :, place(ctx + p)[1]].copy() for p in path]
    for i, row in enumerate(rows):
        if row is not None and path[i] != i and place(ctx + i) is not None:
            at, line = place(ctx + i)
            pool[:, at, :, line] = row


def beam(logits, scores, n):
    """(best, parents, tokens), each ``[items, n]``; ``logits [items, beams, V]``."""
    items, beams, V = logits.shape
    best, parents, tokens = np.empty((items, n)), np.empty((items, n), dtype=int), np.empty((items, n), dtype=int)
    for i in range(items):
        value = np.full((beams, V), -math.inf)
        for w in range(beams):
            x = logits[i, w].astype(np.float64)
            if not math.isfinite(scores[i, w]) or not (x < math.inf).all() or not (x > -math.inf).any():
                continue
            top = x.max()
            value[w] = float(scores[i, w]) + (x - (top + math.log(np.exp(x - top).sum())))
        flat = value.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:n]
        best[i], parents[i], tokens[i] = flat[order], order // V, order % V
    return best, parents, tokens


def copy(array, source, target, dim):
    """Entries along ``dim``: all read before any is written, the last copy to a target counts."""
    old = np.moveaxis(array, dim, 0).copy()
    new = np.moveaxis(array, dim, 0)
    for a, b in zip(source, target):
        if 0 <= a < old.shape[0] and 0 <= b < old.shape[0]:
            new[b] = old[a]
