"""Feed-forward calls at the edges of what their documentation allows, on the GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import TYPES, experts  # noqa: E402, F401 -- a fixture
from test_gpu_feed import problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("f", [2048, 4096, 4100])
@pytest.mark.parametrize("routed", [False, True])
def test_empty_batch_of_a_wide_block(experts, f, routed, dtype):  # noqa: F811
    """No rows through one expert whose sums are long enough to be cut over blocks."""
    s = problem(0, 64, f, 64, 1, 1, dtype, 1)
    m, chosen = (s["gate"], s["up"], s["down"]), s["chosen"] if routed else None
    out, pre = experts.feed(s["x"], *m, chosen, weights=s["weights"], base=s["base"], return_pre=True)
    assert out.shape == (0, 64) and pre.shape == (0, 1, 2, f)
    g = experts.feed_backward(s["grad"], s["x"], *m, chosen, pre, weights=s["weights"], base=s["grad_base"])
    assert g.x.shape == (0, 64) and g.weights.shape == (0, 1)
    assert all(t.shape == s[v].shape and (t == 0).all() for v, t in (("gate", g.gate), ("up", g.up), ("down", g.down)))
