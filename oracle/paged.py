"""float64 definitions of the paged-cache operators (attention, append, eviction).

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  Sequence by sequence, with plain indexing; the int8
codes are taken as the values they stand for (codes times scale).  ``paged_attention`` also returns what the
error bounds of the tests need: the absolute sums that the rounding errors scale with.
"""
from __future__ import annotations

import numpy as np

__all__ = ["gather", "paged_attention", "rope", "kept_tokens"]


def gather(pool: np.ndarray, table_row: np.ndarray, n: int) -> np.ndarray:
    """Tokens [0, n) of one sequence: pool [P, Hkv, page, ...] -> [Hkv, n, ...]."""
    page = pool.shape[2]
    pages = [pool[int(table_row[i])] for i in range(-(-n // page))]
    return np.concatenate(pages, 1)[:, :n] if pages else pool[0][:, :0]


def paged_attention(q, K, V, table, lens):
    """q [B,Hq,D], pools [P,Hkv,page,D] (values, float64) -> dict of

    out [B,Hq,D]; absum [B,Hq,D] = sum p |v|; smax [B,Hq] = max_j sum_i |q_i k_ji| / sqrt(D);
    vmax = max |v|; p: list of [Hq, n] softmax weights.
    """
    q = np.asarray(q, np.float64)
    B, Hq, D = q.shape
    Hkv = K.shape[1]
    G = Hq // Hkv
    r = dict(out=np.zeros((B, Hq, D)), absum=np.zeros((B, Hq, D)), smax=np.zeros((B, Hq)), vmax=0.0, p=[])
    for b in range(B):
        n = int(lens[b])
        p_b = np.zeros((Hq, n))
        if n:
            k, v = gather(K, table[b], n).astype(np.float64), gather(V, table[b], n).astype(np.float64)
            r["vmax"] = max(r["vmax"], float(np.abs(v).max()))
            for h in range(Hq):
                s = k[h // G] @ q[b, h] / np.sqrt(D)
                r["smax"][b, h] = (np.abs(k[h // G]) @ np.abs(q[b, h])).max() / np.sqrt(D)
                e = np.exp(s - s.max())
                p_b[h] = e / e.sum()
                r["out"][b, h] = p_b[h] @ v[h // G]
                r["absum"][b, h] = p_b[h] @ np.abs(v[h // G])
        r["p"].append(p_b)
    return r


def rope(x, cos, sin, positions, axes):
    """x [T, H, D], tables [rows, D/2], positions [A, T], axes [D/2] -> (y, sum of the two absolute products)."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    i = np.arange(half)
    at = np.asarray(positions)[np.asarray(axes)].T  # [T, D/2]
    c, s = np.asarray(cos, np.float64)[at, i][:, None], np.asarray(sin, np.float64)[at, i][:, None]
    lo, hi = x[..., :half], x[..., half:]
    y = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    a = np.concatenate([abs(lo * c) + abs(hi * s), abs(hi * c) + abs(lo * s)], -1)
    return y, a


def kept_tokens(w: np.ndarray, budget: int, recent: int) -> np.ndarray:
    """Indices (ascending) that stay of one (sequence, KV head) with weights w [n], n > budget."""
    n = len(w)
    old = [(-np.inf if np.isnan(x) else -float(x), 0 if np.isnan(x) else 1, j) for j, x in enumerate(w[:n - recent])]
    heavy = sorted(old)[:budget - recent]
    return np.array(sorted(j for _, _, j in heavy) + list(range(n - recent, n)), dtype=np.int64)
