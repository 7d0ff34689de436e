"""float64 numpy restatement of a step of tree-speculative decoding.

Test infrastructure only.  Tree attention: request r's tree nodes are the last
T of its kv_len positions; node i sees every position before the tree and the
nodes j with sees[i, j].  A row that sees nothing is 0 with lse -inf.
"""

from __future__ import annotations

import numpy as np

from .paged_decode import _f64, gather_row_kv


def ancestors(parents):
    """sees[i, j]: node j is node i or an ancestor of it (one tree; parents[i] < i, or -1)."""
    n = len(parents)
    sees = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def tree_request(q, k, v, sees, sm_scale):
    """One request: q [T, Hq, D], k and v [kv_len, Hkv, D], sees [T, T].
    Returns (o [T, Hq, D], lse [T, Hq])."""
    q, k, v = _f64(q), _f64(k), _f64(v)
    n, hq, d = q.shape
    kv_len, hkv, _ = k.shape
    g = hq // hkv
    seen = np.ones((n, kv_len), dtype=bool)
    seen[:, kv_len - n:] = sees
    o, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    for i in range(n):
        at = np.flatnonzero(seen[i])  # masked positions do not enter, whatever they hold
        if at.size == 0:
            continue
        for h in range(hq):
            s = k[at, h // g] @ q[i, h] * sm_scale
            m = s.max()
            p = np.exp(s - m)
            o[i, h] = p @ v[at, h // g] / p.sum()
            lse[i, h] = m + np.log(p.sum())
    return o, lse


def paged_tree(q, cache, qo_indptr, kv_indptr, kv_indices, kv_last, sees, sm_scale=None):
    """Packed q [tokens, Hq, D]; sees: one [T, T] array per request."""
    q = np.asarray(q)
    scale = 1.0 / np.sqrt(q.shape[2]) if sm_scale is None else sm_scale
    o, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    for r in range(len(kv_last)):
        a, e = int(qo_indptr[r]), int(qo_indptr[r + 1])
        if a == e:
            continue
        k, v = gather_row_kv(cache, kv_indptr, kv_indices, kv_last, r)
        o[a:e], lse[a:e] = tree_request(q[a:e], k, v, sees[r], scale)
    return o, lse


def accept(tokens, parents, picks, qo_indptr, max_path):
    """(path, count, kept) of each request, as lists."""
    paths, counts, kept = [], [], []
    for a, e in zip(qo_indptr, qo_indptr[1:]):
        path = [0] if e > a else []
        while path and len(path) < max_path:
            here = path[-1]
            child = next((i for i in range(here + 1, e - a)
                          if parents[a + i] == here and tokens[a + i] == picks[a + here]), None)
            if child is None:
                break
            path.append(child)
        pad = [-1] * (max_path - len(path))
        paths.append(path + pad)
        counts.append(len(path))
        kept.append([int(picks[a + i]) for i in path] + pad)
    return paths, counts, kept


def commit(cache, qo_indptr, kv_indptr, kv_indices, kv_last, path, count):
    """The pool [layers, P, 2, page, Hkv, D] after the accepted paths' tokens moved, one after another."""
    cache = cache.copy()
    ps = cache.shape[3]
    for r in range(len(kv_last)):
        ids = kv_indices[kv_indptr[r]:kv_indptr[r + 1]]
        tree = qo_indptr[r + 1] - qo_indptr[r]
        if len(ids) == 0:
            continue
        base = (len(ids) - 1) * ps + kv_last[r] - tree
        for k in range(min(count[r], len(path[r]))):
            if not k <= path[r][k] < tree:
                break
            s, d = base + path[r][k], base + k
            cache[:, ids[d // ps], :, d % ps] = cache[:, ids[s // ps], :, s % ps]
    return cache
