"""Verification of drafted tokens and low-rank adapters in binary64, straight
from their definitions.

TEST INFRASTRUCTURE ONLY, as pyoracle.
"""
from __future__ import annotations

import numpy as np


def softmax(row, T=1.0):
    """exp((l - max) / T) normalised; T <= 0 or NaN: all on the first maximum;
    NaN and -infinity weigh 0, +infinities share; no candidate: zeros."""
    x = np.asarray(row, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not T > 0:
        return np.eye(1, x.size, int(np.argmax(x)))[0]
    with np.errstate(all="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / T))
    w = np.where(np.isfinite(w), w, 0.0)
    return w / w.sum()


def given(row):
    """Probabilities as given; what is none counts as 0."""
    p = np.asarray(row, np.float64)
    return np.where((p > 0) & np.isfinite(p), p, 0.0)


def draw(r, u):
    """The first index whose running sum is above u times the whole (the last
    one with mass where none is); -1 where the whole is 0."""
    c = np.cumsum(r)
    if not c.size or not c[-1] > 0:
        return -1
    hit = np.flatnonzero((r > 0) & (c > u * c[-1]))
    return int(hit[0]) if hit.size else int(np.flatnonzero(r > 0)[-1])


def at(p, x):
    return float(p[x]) if 0 <= x < p.size else 0.0


def verify(p_rows, q_rows, drafts, u):
    """One sequence: (tokens, acceptance probabilities).  p_rows: n + 1 rows;
    q_rows: n rows, or None for certain drafts."""
    n = len(drafts)
    tokens, accept = [], np.zeros(n)
    for i, x in enumerate(drafts):
        p = at(p_rows[i], x)
        q = 1.0 if q_rows is None else at(q_rows[i], x)
        accept[i] = (1.0 if p >= q else p / q) if p > 0 else 0.0
        if not u[i] * q < p:
            if q_rows is None:
                r = p_rows[i].copy()
                if 0 <= x < r.size:
                    r[x] = 0.0
            else:
                r = np.maximum(p_rows[i] - q_rows[i], 0.0)
            v = draw(r, u[n])
            break
        tokens.append(int(x))
    else:
        i = n
        v = draw(p_rows[n], u[n])
    if v < 0:
        v = max(draw(p_rows[i], u[n]), 0)
    return tokens + [v], accept


def verify_lists(t_lists, d_lists, drafts, u):
    """One sequence against candidate lists: lists are (ids, probabilities,
    kept, token).  (None, None) where a list that counts is not whole."""
    def dist(l):
        ids, probs, kept, token = l
        if kept > len(ids) or (kept <= 0 and token < 0):
            return None
        if kept <= 0:
            return np.array([token]), np.array([1.0])
        w = given(probs[:kept])
        return np.asarray(ids[:kept]), w / w.sum() if w.sum() > 0 else w

    n = len(drafts)
    tokens, accept = [], np.zeros(n)
    for i in range(n + 1):
        t = dist(t_lists[i])
        d = dist(d_lists[i]) if d_lists is not None and i < n else None
        if t is None or (d_lists is not None and i < n and d is None):
            return None, None
        if i == n:
            r = t[1]
            break
        x = drafts[i]
        p = float(t[1][t[0] == x].sum())
        q = 1.0 if d_lists is None else float(d[1][d[0] == x].sum())
        accept[i] = (1.0 if p >= q else p / q) if p > 0 else 0.0
        if u[i] * q < p:
            tokens.append(int(x))
            continue
        if d_lists is None:
            r = np.where(t[0] == x, 0.0, t[1])
        else:
            share = dict(zip(d[0].tolist(), d[1].tolist()))
            r = np.array([max(a - share.get(v, 0.0), 0.0) for v, a in zip(t[0].tolist(), t[1].tolist())])
        break
    v = draw(r, u[n])
    if v < 0:
        v = max(draw(t[1], u[n]), 0)
    return tokens + [int(t[0][v])], accept


def append(tokens, history, done, stop_ids):
    """What a decode loop keeps of a step's tokens: (kept tokens, done)."""
    if done:
        return [], True
    for i, t in enumerate(tokens):
        if t in stop_ids:
            return tokens[:i + 1], True
        history.append(t)
    return tokens, False


def lora(x, a, b, scales, ranks, slots, base):
    """(y, bound): y = base + scale (x A^T) B^T in binary64, and what any
    order of binary32 sums stays within: every product and sum of a term rounds
    by at most 2^-24 of the sum of magnitudes, K + rank + 6 times on its way."""
    M, K, N = x.shape[0], x.shape[1], b.shape[1]
    y = np.zeros((M, N)) if base is None else base.astype(np.float64).copy()
    mag = np.abs(y)
    x = x.astype(np.float64)
    for m in range(M):
        s = int(slots[m])
        if not 0 <= s < a.shape[0]:
            continue
        r = min(max(int(ranks[s]), 0), a.shape[1])
        A, B = a[s, :r].astype(np.float64), b[s, :, :r].astype(np.float64)
        sc = float(scales[s])
        y[m] += sc * (B @ (A @ x[m]))
        mag[m] += abs(sc) * (np.abs(B) @ (np.abs(A) @ np.abs(x[m])))
    return y, (K + a.shape[1] + 6) * 2.0 ** -24 * mag + 1e-37
