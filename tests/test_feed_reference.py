"""The references of the feed-forward, dropout and log-probability operators: gradients against
differences, and the generator against its published vectors."""

from __future__ import annotations

import feed_reference as ref
import numpy as np
import pytest


@pytest.mark.parametrize("name", ["silu", "gelu", "relu"])
def test_feed_gradient_is_its_difference(name):
    rng = np.random.default_rng(3)
    n, d, f, o, a, k = 5, 4, 3, 6, 3, 2
    v = dict(x=rng.standard_normal((n, d)), gate=rng.standard_normal((a, f, d)), up=rng.standard_normal((a, f, d)), down=rng.standard_normal((a, o, f)),
             weights=rng.random((n, k)))
    chosen = np.array([[0, 2], [2, -1], [1, 1], [7, 0], [-1, -1]])
    grad = rng.standard_normal((n, o))

    def value():
        return float((ref.feed(v["x"], v["gate"], v["up"], v["down"], chosen, v["weights"], name=name)["out"][0] * grad).sum())

    got = ref.feed(v["x"], v["gate"], v["up"], v["down"], chosen, v["weights"], name=name, grad=grad)
    h = 1e-6  # truncation h^2, rounding 2^-53 / h: under 1e-8 here
    for key in v:
        flat, g = v[key].reshape(-1), got[key][0].reshape(-1)
        for i in range(flat.size):
            keep = flat[i]
            flat[i] = keep + h
            hi = value()
            flat[i] = keep - h
            lo = value()
            flat[i] = keep
            assert abs((hi - lo) / (2 * h) - g[i]) < 1e-7, (key, i)


def test_rate_gradient_is_its_difference():
    rng = np.random.default_rng(4)
    z = rng.standard_normal((6, 9)) * 2
    z[rng.random(z.shape) < 0.2] = -np.inf
    t = np.array([0, 3, -100, 8, 9, 2])
    glp, gent, glse = rng.standard_normal((3, 6))
    lp, ent, lse, _, _, p, logp = ref.rate(z, t, 0)
    dz, _ = ref.rate_backward(p, logp, ent, t, glp, gent, glse)

    def value(zz):
        a, b, c = ref.rate(zz, t, 0)[:3]
        return float((np.where(np.isfinite(a), a, 0.0) * glp + b * gent + c * glse).sum())

    h = 1e-6
    for i in range(6):
        for j in range(9):
            if z[i, j] == -np.inf:
                assert dz[i, j] == 0
                continue
            hi, lo = z.copy(), z.copy()
            hi[i, j] += h
            lo[i, j] -= h
            assert abs((value(hi) - value(lo)) / (2 * h) - dz[i, j]) < 1e-7


def test_philox_is_the_published_one():
    """The known answers of the generator's authors for a zero counter and key, and a count of its words."""
    assert [int(w) for w in ref.words(4, 0, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    w = ref.words(4000, 12345, 6, 7)
    for p in (0.1, 0.5, 0.9):  # 4,000 draws: five standard deviations
        assert abs(float((w >= round(p * 2**32)).mean()) - (1 - p)) < 5 * (p * (1 - p) / 4000) ** 0.5
