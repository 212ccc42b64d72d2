"""Feed-forward blocks, dropout and log probabilities in 64 bits on the CPU, straight from their
formulas, and how far results with roundings at known places may be from them.

u = 2^-24 is the rounding of fp32; HALF that of a type (half a step: 2^-8 bf16, 2^-11 fp16, u fp32) and STEP the
smallest step of fp16, below which its rounding is absolute."""

from __future__ import annotations

import math

import numpy as np

U = 2.0**-24
HALF = {"fp32": U, "bf16": 2.0**-8, "fp16": 2.0**-11}
STEP = {"fp32": 2.0**-140, "bf16": 2.0**-133, "fp16": 2.0**-24}

_erf = np.vectorize(math.erfc, otypes=[float])


def act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        t = np.where(g > 0, 1 / (1 + np.exp(-np.abs(g))), np.exp(-np.abs(g)) / (1 + np.exp(-np.abs(g))))
        return g * t, t * (1 + g * (1 - t))
    if name == "gelu":
        c = 0.5 * _erf(-g / math.sqrt(2)) if g.size else g
        return g * c, c + g * np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return np.maximum(g, 0), (g > 0).astype(float)


def feed(x, gate, up, down, chosen, weights=None, base=None, name="silu", dtype="fp32", grad=None, grad_base=None):
    """A dict of every result with its bound: out, pre [n, k, 2, f] and, with grad, x, gate, up, down, weights.

    Where the bounds come from: a sum of m products is off by (m + 8) u times its magnitude in any order;
    an activation by 16 u of its value (exp, a sum, a quotient, a product; erfc likewise) and its derivative
    by 16 u (1 + |g|); both pass an error of g on by at most 1.13 and, the derivative, 1.0 (relu's derivative
    jumps: there the whole term where g is 0 within its error).  The hidden vector, weighted, and the gradients of g
    and u are rounded to the type once (HALF, STEP) before the second products, every result once at its end."""
    half, step = HALF[dtype], STEP[dtype]
    n, d = x.shape
    a, f, _ = gate.shape
    o, k = down.shape[1], chosen.shape[1]
    w = np.ones((n, k)) if weights is None else weights
    out = np.zeros((n, o)) if base is None else base.copy()
    oute = np.zeros((n, o))
    pre, pree = np.zeros((n, k, 2, f)), np.zeros((n, k, 2, f))
    r = dict()
    if grad is not None:
        dx = np.zeros((n, d)) if grad_base is None else grad_base.copy()
        dxe = np.zeros((n, d))
        dm = [np.zeros(gate.shape), np.zeros(up.shape), np.zeros(down.shape)]
        dme = [np.zeros(gate.shape), np.zeros(up.shape), np.zeros(down.shape)]
        dw, dwe = np.zeros((n, k)), np.zeros((n, k))
    for q in range(a):
        i, j = np.nonzero(chosen == q)
        if not len(i):
            continue
        P, Q, R, X, W = gate[q], up[q], down[q], x[i], w[i, j][:, None]
        aP, aQ, aR, aX, aW = (np.abs(v) for v in (P, Q, R, X, W))
        g, u = X @ P.T, X @ Q.T
        ge, ue = (d + 8) * U * (aX @ aP.T), (d + 8) * U * (aX @ aQ.T)
        s, t = act(g, name)
        se = 16 * U * np.abs(s) + 1.13 * ge + 2.0**-120
        hid = s * u
        hide = se * np.abs(u) + np.abs(s) * ue + se * ue + 2 * U * np.abs(hid)
        h = W * hid
        he = aW * hide + 2 * U * np.abs(h)
        he = he + half * (np.abs(h) + he) + step
        pre[i, j, 0], pre[i, j, 1] = g, u
        pree[i, j, 0], pree[i, j, 1] = ge, ue
        np.add.at(out, i, h @ R.T)
        np.add.at(oute, i, he @ aR.T + (f + k + 8) * U * ((np.abs(h) + he) @ aR.T))
        if grad is None:
            continue
        G = grad[i]
        e = G @ R
        ee = (o + 8) * U * (np.abs(G) @ aR)
        dw[i, j] = (e * hid).sum(1)
        dwe[i, j] = (ee * np.abs(hid) + np.abs(e) * hide + ee * hide).sum(1) + (f + 40) * U * (np.abs(e * hid) + ee * hide).sum(1)
        te = 16 * U * (1 + np.abs(g)) + ge
        if name == "relu":
            te = np.where(np.abs(g) <= ge, 1.0, 0.0)
        dg, du = W * e * u * t, W * e * s
        dge = aW * (ee * np.abs(u * t) + np.abs(e) * (ue * np.abs(t) + np.abs(u) * te + ue * te) + ee * (ue * np.abs(t) + np.abs(u) * te)) + 8 * U * np.abs(dg)
        due = aW * (ee * np.abs(s) + np.abs(e) * se + ee * se) + 8 * U * np.abs(du)
        dge = dge + half * (np.abs(dg) + dge) + step
        due = due + half * (np.abs(du) + due) + step
        gm, um = np.abs(dg) + dge, np.abs(du) + due
        np.add.at(dx, i, dg @ P + du @ Q)
        np.add.at(dxe, i, dge @ aP + due @ aQ + (2 * f + k + 8) * U * (gm @ aP + um @ aQ))
        c = len(i) + 24  # up to 16 parts of the sum
        aG = np.abs(G)
        for v, ve, (l, le, m) in zip(dm, dme, ((dg, dge, X), (du, due, X), (G, None, None))):
            if m is None:
                v[q] = G.T @ h
                ve[q] = aG.T @ he + c * U * (aG.T @ (np.abs(h) + he))
            else:
                v[q] = l.T @ m
                ve[q] = le.T @ np.abs(m) + c * U * ((np.abs(l) + le).T @ np.abs(m))

    def rounded(v, e):
        return v, e + half * (np.abs(v) + e) + step + 2 * U * np.abs(v)

    r["out"], r["pre"] = rounded(out, oute), (pre, pree + 2.0**-140)
    if grad is not None:
        r["x"], r["weights"] = rounded(dx, dxe), (dw, dwe + 2.0**-140)
        r["gate"], r["up"], r["down"] = (rounded(v, e) for v, e in zip(dm, dme))
    return r


# ---- dropout ----


def words(count, seed, step, site):
    """Philox4x32-10 in Python's whole numbers: `count` words from counter 0 on."""
    got = []
    for b in range(-(-count // 4)):
        c = [b & 0xFFFFFFFF, b >> 32, site, step & 0xFFFFFFFF]
        k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(q >> 32) ^ c[1] ^ k0, q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k1, p & 0xFFFFFFFF]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        got += c
    return np.array(got[:count], dtype=np.uint64)


# ---- log probabilities ----


def rate(z, targets, k):
    """z [n, v]: log_probs, entropy, lse, top, top_log_probs and p."""
    n, v = z.shape
    lp, ent, lse = np.zeros(n), np.zeros(n), np.full(n, -np.inf)
    top, toplp, p = np.full((n, k), -1, np.int64), np.full((n, k), -np.inf), np.zeros((n, v))
    logp = np.full((n, v), -np.inf)
    for i in range(n):
        ok = np.flatnonzero(z[i] > -np.inf)  # False for NaN
        if len(ok):
            m = z[i, ok].max()
            if m == np.inf:
                lse[i], ent[i], logp[i] = np.inf, np.nan, np.nan
            else:
                log_s = np.log(np.exp(z[i, ok] - m).sum())
                lse[i] = m + log_s
                logp[i, ok] = (z[i, ok] - m) - log_s  # an m of 1e38 leaves nothing of log_s in lse
                p[i, ok] = np.exp(logp[i, ok])
                ent[i] = -(p[i, ok] * logp[i, ok]).sum()
            order = ok[np.argsort(-z[i, ok], kind="stable")][:k]
            top[i, : len(order)] = order
            toplp[i, : len(order)] = logp[i, order]
        if 0 <= targets[i] < v:
            lp[i] = logp[i, targets[i]]
    return lp, ent, lse, top, toplp, p, logp


def rate_backward(p, logp, ent, targets, glp, gent, glse):
    """dz and the magnitude that it is made of."""
    n, v = p.shape
    has = (targets >= 0) & (targets < v)
    g = np.where(has, glp, 0.0)
    l = np.where(p > 0, logp, 0.0)
    dz = p * ((glse - g - gent * ent)[:, None] - gent[:, None] * l)
    mag = p * ((np.abs(glse) + np.abs(g) + np.abs(gent * ent))[:, None] + np.abs(gent[:, None] * l))
    rows = np.flatnonzero(has)
    on = logp[rows, targets[rows]] > -np.inf
    dz[rows[on], targets[rows[on]]] += g[rows[on]]
    mag[rows[on], targets[rows[on]]] += np.abs(g[rows[on]])
    return dz, mag
