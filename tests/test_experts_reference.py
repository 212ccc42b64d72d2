"""The references of the routing tests against each other."""

from __future__ import annotations

import experts_reference as ref
import experts_wide_reference as wide
import numpy as np
import pytest


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (40, 7, 3), (25, 30, 16), (3, 5, 5)])
def test_rows_at_once_are_rows_one_by_one(n, e, k, masked, normalize):
    rng = np.random.default_rng(n)
    z = np.round(rng.standard_normal((n, e)) * 2) / 2  # ties
    z[rng.random((n, e)) < 0.2] = -np.inf
    z[rng.random((n, e)) < 0.1] = np.nan
    if n > 3:
        z[n // 2] = -np.inf
    mask = rng.random(n) < 0.7 if masked else None
    a, b = ref.route(z, k, mask, normalize), wide.route(z, k, mask, normalize)
    for x, y in zip(a, b):
        np.testing.assert_allclose(x, y, rtol=1e-12, atol=1e-14)
    w, ex, counts, _, rows, _, p = a
    dw = rng.standard_normal((n, k))
    for x, y in zip(ref.route_backward(p, w, ex, counts, rows, dw, 0.7, normalize), wide.route_backward(p, w, ex, counts, rows, dw, 0.7, normalize)):
        np.testing.assert_allclose(x, y, rtol=1e-12, atol=1e-14)
