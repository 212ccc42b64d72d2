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


def test_gradients_of_no_rows(experts):  # noqa: F811
    """The sum of an empty batch's results: nothing for the rows, 0 for what all rows share."""
    s = problem(0, 64, 48, 64, 3, 2, "bf16", 1)
    x, base, gate = (s[v].clone().requires_grad_() for v in ("x", "base", "gate"))
    y = experts.fed(x, gate, s["up"], s["down"], s["chosen"], weights=s["weights"], base=base)
    y = experts.dropped(y, 0.1, torch.tensor([1, 2], device="cuda"), base=base)
    low = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
    experts.adapted(y, low, low.detach(), s["chosen"][:, 0]).sum().backward()
    assert x.grad.shape == base.grad.shape == (0, 64) and (gate.grad == 0).all() and (low.grad == 0).all()
    z = torch.zeros(0, 64, device="cuda", requires_grad=True)
    r = experts.rated(z, s["chosen"][:, 0])
    (r.log_probs.sum() + r.entropy.sum() + experts.routed(z, 2).weights.sum()).backward()
    assert z.grad.shape == (0, 64)
