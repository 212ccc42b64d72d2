"""Routing and adapters in 64 bits on the CPU, straight from their formulas, row by row
where the operator is defined row by row.  With every result comes the sum of the
magnitudes it is made of, which the tests' rounding bounds are multiples of."""

from __future__ import annotations

import numpy as np


def route(z, k, mask=None, normalize=False):
    """z [n, e] float64.  Returns weights, experts, counts, prob_sums, rows, loss, p."""
    n, e = z.shape
    w, ex, p = np.zeros((n, k)), np.full((n, k), -1, np.int64), np.zeros((n, e))
    counts, rows = np.zeros(e, np.int64), 0
    for i in range(n):
        if mask is not None and not mask[i]:
            continue
        ok = [j for j in range(e) if z[i, j] > -np.inf]  # False for NaN too
        if not ok:
            continue
        rows += 1
        m = max(z[i, j] for j in ok)
        p[i, ok] = np.exp(z[i, ok] - m)
        p[i] /= p[i].sum()
        top = sorted(ok, key=lambda j: (-z[i, j], j))[:k]
        ex[i, : len(top)] = top
        w[i, : len(top)] = p[i, top]
        if normalize:
            w[i] /= w[i].sum()
        counts[top] += 1
    sums = p.sum(0)
    loss = e / (k * rows * rows) * float((counts * sums).sum()) if rows else 0.0
    return w, ex, counts, sums, rows, loss, p


def route_backward(p, w, ex, counts, rows, dw, dloss, normalize):
    """Returns dz [n, e] and the magnitudes it is made of."""
    n, e = p.shape
    k = ex.shape[1]
    G = np.zeros((n, e))
    if rows:
        G += dloss * e / (k * rows * rows) * counts
    gate = np.zeros((n, e))
    gate_mag = np.zeros((n, e))
    for i in range(n):
        on = ex[i] >= 0
        d = np.where(on, dw[i], 0.0)
        inner = float((w[i] * d).sum())
        inner_mag = float(np.abs(w[i] * d).sum())
        if normalize:
            gate[i, ex[i][on]] += (w[i] * (d - inner))[on]
            gate_mag[i, ex[i][on]] += (np.abs(w[i]) * (np.abs(d) + inner_mag))[on]
        else:
            gate[i, ex[i][on]] += (w[i] * d)[on]
            gate[i] -= p[i] * inner
            gate_mag[i, ex[i][on]] += np.abs(w[i] * d)[on]
            gate_mag[i] += p[i] * inner_mag
    dz = p * (G - (p * G).sum(1, keepdims=True)) + gate
    mag = p * (np.abs(G) + (p * np.abs(G)).sum(1, keepdims=True)) + gate_mag
    return dz, mag


def _factors(ids, a, gates, scales):
    has = (ids >= 0) & (ids < a)
    f = np.zeros(len(ids))
    f[has] = (scales[ids[has]] if scales is not None else 1.0) * (gates[has] if gates is not None else 1.0)
    return has, f


def adapt(x, down, up, ids, base=None, gates=None, scales=None):
    """Returns out, low and the magnitudes of out's adapter part."""
    n, a, r, o = x.shape[0], down.shape[0], down.shape[1], up.shape[2]
    has, f = _factors(ids, a, gates, scales)
    out = np.zeros((n, o)) if base is None else base.copy()
    low, mag = np.zeros((n, r)), np.zeros((n, o))
    for q in range(a):
        i = np.flatnonzero(has & (ids == q))
        low[i] = x[i] @ down[q].T
        out[i] += f[i, None] * (low[i] @ up[q])
        mag[i] = np.abs(f[i, None]) * ((np.abs(x[i]) @ np.abs(down[q]).T) @ np.abs(up[q]))
    return out, low, mag


def adapt_backward(dy, x, down, up, ids, base=None, gates=None, scales=None):
    """Returns (dx, ddown, dup, dgates) and the magnitudes of each (dx's without base)."""
    n, a = x.shape[0], down.shape[0]
    has, f = _factors(ids, a, gates, scales)
    dx = np.zeros(x.shape) if base is None else base.copy()
    dA, dB, dg = np.zeros(down.shape), np.zeros(up.shape), np.zeros(n)
    mx, mA, mB, mg = np.zeros(x.shape), np.zeros(down.shape), np.zeros(up.shape), np.zeros(n)
    for q in range(a):
        i = np.flatnonzero(has & (ids == q))
        A, B, s = down[q], up[q], 1.0 if scales is None else scales[q]
        t, u, c = x[i] @ A.T, dy[i] @ B.T, f[i, None]
        tm, um, cm = np.abs(x[i]) @ np.abs(A).T, np.abs(dy[i]) @ np.abs(B).T, np.abs(c)
        dx[i] += c * (u @ A)
        dA[q], dB[q] = (c * u).T @ x[i], (c * t).T @ dy[i]
        dg[i] = s * (t * u).sum(1)
        mx[i] = cm * (um @ np.abs(A))
        mA[q], mB[q] = (cm * um).T @ np.abs(x[i]), (cm * tm).T @ np.abs(dy[i])
        mg[i] = np.abs(s) * (tm * um).sum(1)
    return (dx, dA, dB, dg), (mx, mA, mB, mg)
