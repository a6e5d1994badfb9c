"""The page-bounds, page-selection, chosen-page attention and draft-verification operators from their
definitions, in 64 bits on the CPU: what the kernels' tests compare with."""
from __future__ import annotations

import math

import numpy as np


def least_power(a):
    """The least power of two from 2^-126 on with a <= 127 times it (a >= 0, finite)."""
    e = -126
    while e < 127 and a > 127.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def page_bounds(keys):
    """(hi, lo, scale) of keys [n][D]."""
    keys = np.asarray(keys, np.float64)
    if not np.isfinite(keys).all():
        return np.full(keys.shape[1], 127), np.full(keys.shape[1], -127), np.inf
    s = least_power(np.abs(keys).max())
    return np.ceil(keys.max(0) / s), np.floor(keys.min(0) / s), s


def update_bounds(bounds, scale, key_at, table, start, n, P, H, pages):
    """In place, for one sequence; key_at(page, head, count) gives the page's first keys."""
    for p in range(start // P, (start + n - 1) // P + 1):
        if p >= len(table) or not 1 <= table[p] <= pages:
            continue
        i = table[p] - 1
        for h in range(H):
            hi, lo, s = page_bounds(key_at(i, h, min(P, start + n - p * P)))
            bounds[i, h, 0], bounds[i, h, 1], scale[i, h] = hi, lo, s


def select(q, bounds, scale, table, last, P, keep, sinks, window):
    """(page ids, keys) of one token that sees positions 0 .. last; q [Hq][D] float64."""
    H = bounds.shape[1]
    G = q.shape[0] // H
    seen = min(last // P + 1, len(table))
    ids = np.clip(np.asarray(table[:seen]) - 1, 0, bounds.shape[0] - 1)
    tables, lengths = np.zeros((H, keep), np.int32), np.zeros(H, np.int32)
    for h in range(H):
        best = np.full(seen, -np.inf)
        for g in range(G):
            row = q[h * G + g]
            if np.isfinite(row).all():
                s = least_power(np.abs(row).max())
                w = np.rint(row / s)
            else:
                s, w = 2.0 ** -126, np.zeros_like(row)
            hi, lo = bounds[ids, h, 0].astype(np.float64), bounds[ids, h, 1].astype(np.float64)
            best = np.maximum(best, np.where(w > 0, w * hi, w * lo).sum(1) * s)
        with np.errstate(invalid="ignore"):
            score = best * scale[ids, h].astype(np.float64)
        score[np.isnan(score)] = np.inf
        index = np.arange(seen)
        forced = (index < sinks) | (index >= seen - window)
        order = sorted(range(seen), key=lambda i: (not forced[i], -score[i], i))
        kept = sorted(order[:keep])
        tables[h, :len(kept)] = [table[i] for i in kept]
        lengths[h] = (len(kept) - 1) * P + min(last + 1 - (seen - 1) * P, P)
    return tables, lengths


def attend(q, keys, values, scale):
    """Rows q [G][D] over keys and values [n][D]: (output, sum p |v|, largest sum |q k| scale)."""
    if len(keys) == 0:
        z = np.zeros((q.shape[0], q.shape[1]))
        return z, z, 0.0
    s = q @ keys.T * scale
    size = (np.abs(q) @ np.abs(keys).T * scale).max()
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return p @ values, p @ np.abs(values), size


def verify(x, p, q, u, n):
    """(accepted, tokens [N + 1]) of one sequence: x [N], p [N + 1][V], q [N][V] or None, u [N + 1], n drafts."""
    N, V = len(x), p.shape[1]
    p = p.astype(np.float64)
    q = None if q is None else q.astype(np.float64)
    u = u.astype(np.float64)
    n = min(max(n, 0), N)
    a = 0
    while a < n and 0 <= x[a] < V and u[a] * (1.0 if q is None else q[a, x[a]]) < p[a, x[a]]:
        a += 1

    def mass(w):
        w = w.copy()
        w[~(np.isfinite(w) & (w > 0))] = 0
        return w

    w = p[a].copy()
    if a < n:
        if q is not None:
            with np.errstate(invalid="ignore"):
                w = w - q[a]
        elif 0 <= x[a] < V:
            w[x[a]] = 0
    w = mass(w)
    if not w.any():
        w = mass(p[a])
    token = -1
    if w.any():
        c = np.cumsum(w)
        hit = np.nonzero((w > 0) & (c > u[N] * c[-1]))[0]
        token = int(hit[0]) if len(hit) else int(np.nonzero(w)[0][-1])
    return a, [int(x[i]) if i < a else (token if i == a else -1) for i in range(N + 1)]


def finite_sum_error(D, keys):
    """Bounds used by the tolerances: relative error of a float sum of D products (each product and each
    addition rounds once) and of one over `keys` terms."""
    return (D + 1) * 2.0 ** -24, (keys + 1) * 2.0 ** -24


def attention_tolerance(out, weight, size, D, keys, p_eps, out_eps):
    """Per element. Scores are float sums, off by at most ds = (D + 1) 2^-24 sum |q k| scale + one more
    rounding; a weight then by a factor e^(2 ds) and by p_eps (its rounding before the value product) and
    the exponential's own error (2^-21 of its argument's range, |x| < 2^7 in base 2, and one unit); sums
    over the keys add (keys + 1) 2^-24 twice (products and the sum of weights); the output rounds once."""
    sum_d, sum_k = finite_sum_error(D, keys)
    ds = (sum_d + 2.0 ** -23) * size
    rel = math.expm1(2 * ds) + p_eps + 2.0 ** -20 + 2 * sum_k
    return rel * weight * 1.01 + out_eps * np.abs(out) * 1.01 + 1e-30
