"""The drafted-token operators from their definitions, in 64 bits, for the tests."""
import numpy as np


def path_of(parents, i):
    """Node i's ancestors and itself, first to last."""
    path = []
    while i >= 0:
        path.append(i)
        i = parents[i]
    return path[::-1]


def attention_tree(q, k, v, prefix, parents, window=0):
    """q [nodes, heads, hd], k/v [prefix + nodes, hd] -> [nodes, heads, hd]."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    y = np.empty_like(q)
    for i in range(len(parents)):
        path = path_of(parents, i)
        pos = prefix + len(path) - 1
        first = max(0, pos - window + 1) if window else 0
        rows = list(range(first, prefix)) + [prefix + j for d, j in enumerate(path)
                                             if prefix + d >= first]
        s = q[i] @ k[rows].T
        p = np.exp(s - s.max(1, keepdims=True))
        y[i] = (p @ v[rows]) / p.sum(1, keepdims=True)
    return y


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(ids, p): the tokens that the cuts leave, in index order, and their e^d."""
    t, top_p, min_p = (float(np.float32(a)) for a in (temperature, top_p, min_p))
    x = x.astype(np.float64)
    ids = np.flatnonzero(np.isfinite(x))
    if not ids.size:
        return ids, np.empty(0)
    ids = ids[np.argsort(-x[ids], kind="stable")]
    if t == 0:
        return ids[:1], np.ones(1)
    if top_k:
        ids = ids[:top_k]
    d = (x[ids] - x[ids[0]]) / t
    p = np.exp(d)
    n = len(ids)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(p)[:-1]])
        n = int((before < top_p * p.sum()).sum())
    if min_p > 0:  # p >= min_p, without rounding p (e^-1e-45 is below 1)
        n = min(n, int((d >= np.log(min_p)).sum()))
    order = np.argsort(ids[:n])
    return ids[:n][order], p[:n][order]


def sample(x, u, **cuts):
    """(token, probability) of one row."""
    ids, p = kept(x, **cuts)
    if not ids.size:
        return -1, 0.0
    u = 0.0 if not u > 0 else float(u)
    upto = np.cumsum(p)
    at = min(int((upto <= u * upto[-1]).sum()), len(ids) - 1)
    return int(ids[at]), p[at] / upto[-1]
