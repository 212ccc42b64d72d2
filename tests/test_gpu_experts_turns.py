"""The kernels' loops past their first turn, and the instances that only large calls reach.
Shapes are worked out from the launch rules beside each test; bounds are those of
test_gpu_experts."""

from __future__ import annotations

import math

import experts_wide_reference as ref
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import HALF, STEP, TYPES, U, check_adapt, experts, f64, near, problem, scores  # noqa: E402, F401 -- a fixture

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


# ---- route: 768 blocks of four waves take a group of rows each at once (twice that backward for 33 to 64
# experts); a group has 64 rows up to 32 experts, 8 up to 256, 4 up to 512, one beyond ----

WAVES = 768 * 4


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,e,k", [(200_003, 8, 2), (400_010, 29, 1), (50_003, 40, 3), (55_001, 64, 16), (24_999, 200, 5), (52_345, 256, 8), (13_001, 300, 7),
                                   (27_002, 512, 2), (7_001, 700, 16), (9_999, 2048, 4)])
def test_route_waves_take_several_groups(experts, n, e, k, dtype):  # noqa: F811
    """A wave's second and third groups of rows: scores loaded ahead, column sums and counts
    that go on, gates of one group cleared before the next.  Gates that were left would show
    at the experts that the earlier rows took."""
    print("route turns", n, e, k, dtype, flush=True)
    rows_a_group = 64 if e <= 32 else 8 if e <= 256 else 4 if e <= 512 else 1
    turns = math.ceil(math.ceil(n / rows_a_group) / WAVES)
    assert turns > 1
    g = torch.Generator().manual_seed(n)
    z = scores(n, e, "normal", TYPES[dtype], n)
    z[torch.rand(n, e, generator=g) < 0.02] = -math.inf
    mask = torch.rand(n, generator=g) < 0.9
    normalize = k % 2 == 0
    dw, dl = torch.randn(n, k, generator=g), 0.3 * n
    want = ref.route(f64(z), k, mask.numpy(), normalize)
    w, ex, counts, sums, rows, loss, p = want
    z, mask, dw = z.cuda(), mask.cuda(), dw.cuda()
    r = experts.route(z, k, mask=mask, normalize=normalize)
    again = experts.route(z, k, mask=mask, normalize=normalize)
    for a, b in zip(r, again):
        assert torch.equal(a, b)
    finite = f64(z)[np.isfinite(f64(z))]
    rel = 2 * (2 * (finite.max() - finite.min()) + math.log2(e) + 16) * U
    np.testing.assert_array_equal(r.experts.cpu().numpy(), ex)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), counts)
    assert r.rows.tolist() == [rows]
    near(r.weights, w, rel * w + 2.0**-120, "weights")
    # a column's sum: a wave's turns, its lanes' log2 64 and the waves' four in fp32, then fp64
    near(r.prob_sums, sums, (rel + (turns + 6 + 4 + 8) * U) * sums + 2.0**-120, "prob_sums")
    near(r.loss, np.float64(loss), (rel + (turns + 6 + 4 + 8) * U) * loss, "loss")
    for dw_, dl_ in ((dw, dl), (dw, None), (None, dl)):
        got = experts.route_backward(z, r, grad_weights=dw_, grad_loss=None if dl_ is None else torch.tensor(dl_, device="cuda"), mask=mask, normalize=normalize)
        want, mag = ref.route_backward(p, w, ex, counts, rows, np.zeros((n, k)) if dw_ is None else f64(dw_), dl_ or 0.0, normalize)
        near(got, want, 2 * (rel + (e + k + 8) * U) * mag + HALF[dtype] * np.abs(want) + STEP[dtype] + 2.0**-120, "grad_logits")


# ---- adapt: a tile has 64, 32 or 16 rows, the most that leave tiles times stretches of columns (512 of a
# 16-bit type, 256 of fp32; of d and o together) at 1,536; a tile's columns go to ceil(1,024 / tiles) blocks ----


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("r", [12, 30, 64, 100])
def test_adapt_large_tiles_and_second_stretches(experts, r, dtype):  # noqa: F811
    """64-row tiles (516 of them), two blocks for the three stretches of a row in both
    directions, and 512-row chunks, in which the rows by rows take several turns."""
    print("adapt 64-row tiles", r, dtype, flush=True)
    d, o = (1032, 1040) if dtype != "fp32" else (520, 600)
    check_adapt(experts, problem(33_001, d, o, r, 5, dtype, r), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,wide,narrow,r,a", [(16_401, 1032, 40, 20, 70), (16_401, 1032, 40, 100, 3), (3_001, 4100, 520, 64, 7), (3_001, 4100, 520, 9, 40)])
def test_adapt_small_tiles_and_second_stretches(experts, n, wide, narrow, r, a, dtype):  # noqa: F811
    """32- and 16-row tiles whose blocks take a second stretch, forward and backward."""
    print("adapt stretches", n, wide, narrow, r, a, dtype, flush=True)
    if dtype == "fp32":
        wide, narrow = wide // 2 + 4, narrow // 2
    check_adapt(experts, problem(n, wide, narrow, r, a, dtype, r), dtype)
    check_adapt(experts, problem(n, narrow, wide, r, a, dtype, r), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_adapt_long_runs_in_large_tiles(experts, dtype):  # noqa: F811
    """One adapter for nearly all rows and none for some: tiles that end where it does."""
    print("adapt long runs", dtype, flush=True)
    d, o = (1032, 520) if dtype != "fp32" else (520, 260)
    s = problem(40_003, d, o, 17, 300, dtype, 5)
    at = torch.arange(40_003)
    s["ids"] = torch.where(at % 11 == 0, -1, torch.where(at < 39_000, 7, at % 300)).int().cuda()
    check_adapt(experts, s, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,r", [(256, 1024, 8), (257, 1024, 8), (128, 1536, 32), (129, 1536, 32), (512, 512, 20), (340, 768, 3), (64, 4096, 9), (65, 4096, 9), (511, 256, 60)])
def test_adapt_few_rows_in_one_turn_and_two(experts, n, d, r, dtype):  # noqa: F811
    """Calls of 256 blocks of one launch, one a CU, and of more."""
    print("adapt one launch", n, d, r, dtype, flush=True)
    check_adapt(experts, problem(n, d, d, r, 7, dtype, n + d), dtype)
