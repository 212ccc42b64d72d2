"""experts_reference's routing for many rows at once."""

from __future__ import annotations

import numpy as np


def route(z, k, mask=None, normalize=False):
    """As experts_reference.route."""
    n, e = z.shape
    ok = z > -np.inf  # False for NaN too
    if mask is not None:
        ok &= mask[:, None]
    z = np.where(ok, z, -np.inf)
    live = ok.any(1)
    p = np.exp(z - np.where(live, z.max(1), 0.0)[:, None])
    p /= np.where(live, p.sum(1), 1.0)[:, None]
    top = np.argsort(-z, axis=1, kind="stable")[:, :k]
    taken = np.take_along_axis(ok, top, 1)
    ex = np.where(taken, top, -1)
    w = np.where(taken, np.take_along_axis(p, top, 1), 0.0)
    if normalize:
        w /= np.where(live, w.sum(1), 1.0)[:, None]
    counts, sums, rows = np.bincount(top[taken], minlength=e), p.sum(0), int(live.sum())
    loss = e / (k * rows * rows) * float((counts * sums).sum()) if rows else 0.0
    return w, ex, counts, sums, rows, loss, p


def route_backward(p, w, ex, counts, rows, dw, dloss, normalize):
    """As experts_reference.route_backward."""
    k, e = ex.shape[1], p.shape[1]
    G = np.broadcast_to(dloss * e / (k * rows * rows) * counts if rows else np.zeros(e), p.shape)
    on = ex >= 0
    d = np.where(on, dw, 0.0)
    inner, inner_mag = (w * d).sum(1, keepdims=True), np.abs(w * d).sum(1, keepdims=True)
    at = (np.nonzero(on)[0], ex[on])
    dz = p * (G - (p * G).sum(1, keepdims=True))
    mag = p * (np.abs(G) + (p * np.abs(G)).sum(1, keepdims=True))
    if normalize:
        np.add.at(dz, at, (w * (d - inner))[on])
        np.add.at(mag, at, (np.abs(w) * (np.abs(d) + inner_mag))[on])
    else:
        np.add.at(dz, at, (w * d)[on])
        np.add.at(mag, at, np.abs(w * d)[on])
        dz -= p * inner
        mag += p * inner_mag
    return dz, mag
