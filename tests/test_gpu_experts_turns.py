"""The kernels' loops past their first turn, and the instances that only large calls reach.
Shapes are worked out from the launch rules beside each test; bounds are those of
test_gpu_experts."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import TYPES, check_adapt, experts, problem  # noqa: E402, F401 -- a fixture

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,a", [(1700, 400), (1700, 9), (9000, 2048)])
def test_adapters_of_several_chunks_among_many(experts, n, a, dtype):  # noqa: F811
    """Adapters of 65, 129 and several hundred rows beside many of one or none: their partial
    sums are apart, wherever their rows start."""
    print("chunks", n, a, dtype, flush=True)
    s = problem(n, 40, 24, 5, a, dtype, n)
    some = [0, a // 3, a // 3 + 1, a // 2, a - 2, a - 1]
    ids = torch.cat([torch.full((c,), q) for q, c in zip(some, (65, 129, 64, n // 4, 1, n // 3))])
    rest = torch.arange(n - len(ids)) % (a + 1)
    g = torch.Generator().manual_seed(n)
    s["ids"] = torch.cat([ids, rest])[torch.randperm(n, generator=g)].int().cuda()
    check_adapt(experts, s, dtype)
