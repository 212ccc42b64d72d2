"""How exactly a low-rank vector enters its bf16 products.

The inputs leave one product in every sum, so nothing but the operator's own roundings is
seen: one nonzero column gives a low-rank value t that is exact in fp32 (a product of two
bf16), and one nonzero rank gives results f t v with v a bf16.  U = 2^-24, the rounding of
fp32.  The roundings are gate times scale (U), times t (U), and the sums of the matrix
cores' products: as many as the low-rank value has parts, each at most 2 U of a sum that
is at most (1 + 2^-8) of the result, however the cores' adder rounds.  Under 16 U in all
for four parts or fewer; then the one rounding to bf16, half a step of the result's own
binade.
"""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import experts, f64  # noqa: E402, F401 -- a fixture

pytestmark = pytest.mark.gpu

U = 2.0**-24


def rounded_once(got, want, what):
    got = f64(got)
    off = np.abs(got - want)
    slack = 16 * U * np.abs(want)
    half_step = np.exp2(np.floor(np.log2(np.maximum(np.abs(want) + slack, 2.0**-100))) - 8)
    bad = ~(off <= half_step + slack)
    if bad.any():
        at = tuple(int(v) for v in np.argwhere(bad)[0])
        pytest.fail(f"{what}: {bad.sum()} of {bad.size} off, first at {at}: {got[at]} for {want[at]}, {(off[at] - half_step[at]) / abs(want[at]) / U:.1f} U past half a step")


def problem(n, narrow, wide, r, a, seed):
    """narrow: [n, narrow] rows with one nonzero column, and the adapters that take them
    with one nonzero rank; wide: dense rows and adapters."""
    g = torch.Generator().manual_seed(seed)
    v = torch.zeros(n, narrow)
    v[:, 1] = torch.randn(n, generator=g)
    A = torch.zeros(a, r, narrow)
    A[:, r // 2, 1] = torch.randn(a, generator=g)
    B = torch.randn(a, r, wide, generator=g)
    dense = torch.randn(n, wide, generator=g)
    v, A, B, dense = (t.bfloat16().cuda() for t in (v, A, B, dense))
    gates, scales = torch.randn(n, generator=g).cuda(), (torch.rand(a, generator=g) + 0.5).cuda()
    ids = torch.arange(n, dtype=torch.int32).cuda() % a
    return v, A, B, dense, gates, scales, ids


# one launch; two launches without a sort; with a sort, every adapter one row
@pytest.mark.parametrize("n,wide,a", [(60, 1000, 50), (100, 4100, 3), (600, 700, 600)])
@pytest.mark.parametrize("r", [5, 20, 40, 100])
def test_bf16_products_round_once(experts, n, wide, a, r):  # noqa: F811
    print("bf16 products", n, wide, a, r, flush=True)
    v, A, B, dense, gates, scales, ids = problem(n, 4, wide, r, a, n + r)
    opt = dict(gates=gates, scales=scales)
    q, t0 = ids.long().cpu().numpy(), r // 2
    f = f64(gates) * f64(scales)[q]
    t = f64(v)[:, 1] * f64(A)[q, t0, 1]
    # forward: v passes down = A and up = B; dU = f t dense
    out, low = experts.adapt(v, A, B, ids, return_low=True, **opt)
    rounded_once(out, (f * t)[:, None] * f64(B)[q, t0], "out")
    g = experts.adapt_backward(dense, v, A, B, ids, low, **opt)
    if a == n:
        rounded_once(g.up[:, t0], (f * t)[:, None] * f64(dense), "grad_up")
    # backward: v as the gradient passes up = A and down = B; dD = f u dense
    _, low = experts.adapt(dense, B, A, ids, return_low=True, **opt)
    g = experts.adapt_backward(v, dense, B, A, ids, low, **opt)
    rounded_once(g.x, (f * t)[:, None] * f64(B)[q, t0], "grad_x")
    if a == n:
        rounded_once(g.down[:, t0], (f * t)[:, None] * f64(dense), "grad_down")
