"""What the Python calls of the routing and adapter operators hand to the library, on CPU
tensors with the library's entry points replaced by a record of their arguments."""

from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def calls(monkeypatch):
    """Calls that reached the library, as (entry point, arguments)."""
    from skmetal_amd import experts

    made = []

    def entry(name):
        return lambda *args: made.append((name, args)) or 0

    names = ("route", "route_backward", "adapt", "adapt_backward")
    monkeypatch.setattr(experts, "_lib", lambda: types.SimpleNamespace(**{f"skmetal_hip_{n}": entry(n) for n in names}))
    monkeypatch.setattr(experts, "_first", lambda t, name: (experts._CODE[t.dtype], t.device))
    monkeypatch.setattr(experts, "_stream", lambda device: None)
    monkeypatch.setattr(experts, "_route_workspace", lambda *sizes: 0)
    monkeypatch.setattr(experts, "_adapt_workspace", lambda *sizes: 0)
    return made


def problem(n=40, d=16, o=24, r=4, a=3):
    return dict(x=torch.zeros(n, d), down=torch.zeros(a, r, d), up=torch.zeros(a, r, o), ids=torch.zeros(n, dtype=torch.int32), grad=torch.zeros(n, o),
                low=torch.zeros(n, r))


APART = {  # rows whose elements do not lie side by side
    "transposed": lambda n, w: torch.zeros(w, n).T,
    "one value a row": lambda n, w: torch.zeros(n, 1).expand(n, w),
    "every other column": lambda n, w: torch.zeros(n, 2 * w)[:, ::2],
}


@pytest.mark.parametrize("how", list(APART))
def test_rows_whose_elements_lie_apart_are_refused(calls, how):
    from skmetal_amd import experts

    s = problem()
    n, d, o = 40, 16, 24
    with pytest.raises(ValueError, match="x's rows .* side by side"):
        experts.adapt(APART[how](n, d), s["down"], s["up"], s["ids"])
    with pytest.raises(ValueError, match="x's rows .* side by side"):
        experts.adapted(APART[how](n, d), s["down"], s["up"], s["ids"])
    with pytest.raises(ValueError, match="grad's rows .* side by side"):
        experts.adapt_backward(APART[how](n, o), s["x"], s["down"], s["up"], s["ids"], s["low"])
    with pytest.raises(ValueError, match="x's rows .* side by side"):
        experts.adapt_backward(s["grad"], APART[how](n, d), s["down"], s["up"], s["ids"], s["low"])
    for option in ("base", "out"):
        with pytest.raises(ValueError, match=f"{option}'s rows .* side by side"):
            experts.adapt(s["x"], s["down"], s["up"], s["ids"], **{option: APART[how](n, o)})
    with pytest.raises(ValueError, match="logits' rows .* side by side"):
        experts.route(APART[how](n, 8), 2)
    assert not calls


def test_rows_apart_keep_their_distance(calls):
    """Wide rows, and one column, whose own stride says nothing."""
    from skmetal_amd import experts

    s = problem()
    experts.adapt(torch.zeros(40, 50)[:, 3:19], s["down"], s["up"], s["ids"])
    one = problem(d=1)
    experts.adapt(torch.zeros(40, 7)[:, :1].T.T, one["down"], one["up"], one["ids"])
    experts.adapt_backward(torch.zeros(40, 60)[:, :24], s["x"], s["down"], s["up"], s["ids"], s["low"])
    assert [c[1][2] for c in calls] == [50, 7, 60]


def test_an_out_in_x_asks_for_the_workspace_of_two_launches(calls, monkeypatch):
    from skmetal_amd import experts

    asked = []
    monkeypatch.setattr(experts, "_adapt_workspace", lambda *sizes: asked.append(sizes[-1]) or 0)
    s = problem(o=16)
    wide = torch.zeros(40, 64)
    for out, call in ((None, 0), (torch.zeros(40, 16), 0), (s["x"], 2), (wide[:, 8:24], 2), (wide[:, 16:32], 2)):
        x = wide[:, :16] if out is not None and out.shape == (40, 16) and out.stride(0) == 64 else s["x"]
        experts.adapt(x, s["down"], s["up"], s["ids"], base=out, out=out)
        assert asked.pop() == call and calls.pop()[0] == "adapt"


def test_routed_results_may_be_changed_in_place(calls):
    from skmetal_amd import experts

    z = torch.zeros(40, 8, requires_grad=True)
    q = experts.routed(z, 2)
    loss = q.loss
    loss.mul_(0.5)
    loss += q.weights.sum()
    for statistic in (q.counts, q.prob_sums, q.rows):
        statistic.add_(1)
    loss.backward()
    assert [c[0] for c in calls] == ["route", "route_backward"] and z.grad.shape == z.shape
    assert q.counts.shape == q.prob_sums.shape == (8,) and q.rows.shape == (1,) and q.loss.shape == ()
    assert q.counts.dtype == q.rows.dtype == torch.int32 and q.prob_sums.dtype == torch.float32


def test_out_is_known_to_autograd(calls):
    """A result in place counts as a change of it: a gradient that needs its old values says
    so, and a tensor on the way of a gradient is refused, since the call records none."""
    from skmetal_amd import experts

    s = problem()
    w = torch.ones(24, requires_grad=True)
    y = torch.zeros(40, 24)
    z = y * w  # keeps y for w's gradient
    experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=y, out=y)
    with pytest.raises(RuntimeError, match="inplace operation"):
        z.sum().backward()
    z = torch.zeros(40, 24) * w
    assert len(calls) == 1
    with pytest.raises(ValueError, match="out requires a gradient"):
        experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=z, out=z)
    assert len(calls) == 1
    with torch.no_grad():
        experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=z, out=z)
    with torch.inference_mode():
        t = torch.zeros(40, 24)
        experts.adapt(s["x"], s["down"], s["up"], s["ids"], out=t)
    assert len(calls) == 3


# ---- the entry points' own checks of places, on addresses that nothing reads ----

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from skmetal_amd import _bridge

    if _bridge._lib is None:
        pytest.fail(f"library not loaded: {_bridge.last_error()}")
    if _bridge.HIP_AVAILABLE:
        pytest.skip("an accepted call would run on these addresses")
    return _bridge._lib


EINVAL, ENODEV = 1, 2


def elements(at, ld, w, n):
    return {at + i * ld + j for i in range(n) for j in range(w)}


def test_out_and_base_share_all_or_nothing(lib):
    """Against the sets of elements themselves: rows in step with each other, out of step,
    crossing, single."""
    import random

    rng = random.Random(5)
    seen = {EINVAL: 0, ENODEV: 0}
    for _ in range(4000):
        n, o = rng.choice([1, 2, 3, 7]), rng.randint(1, 9)
        ld_out = o + rng.choice([0, 1, 5, 12])
        ld_base = rng.choice([ld_out, ld_out, o, rng.randint(0, 25)])
        out, base = rng.randint(0, 60), rng.randint(0, 60)
        code = lib.skmetal_hip_adapt(0, P // 2, 4, P // 4, 8, 4, P // 4, 2 * o, o, P // 8, 1, None, 0, None, P + 4 * base, ld_base, P + 4 * out, ld_out, None, n, 4, o,
                                     2, 1, 4096, 1 << 30, None)
        shared = elements(out, ld_out, o, n) & elements(base, ld_base, o, n)
        fine = not shared or (out == base and (ld_out == ld_base or n == 1))
        assert code == (ENODEV if fine else EINVAL), (n, o, ld_out, ld_base, out, base, lib.skmetal_hip_last_error())
        if not fine:
            assert b"out shares memory with base" in lib.skmetal_hip_last_error()
        seen[code] += 1
    assert min(seen.values()) > 500


def test_out_in_x_needs_the_larger_workspace(lib):
    """64 rows of 4,096 at rank 16 are one launch without scratch, unless out lies in x."""
    sizes = (1, 64, 4096, 4096, 16, 8)
    apart, back, in_x = (lib.skmetal_hip_adapt_workspace(*sizes, call) for call in range(3))
    assert apart == 0 and 0 < in_x and 0 < back

    def adapt(x, out, ld, ws):
        return lib.skmetal_hip_adapt(1, x, ld, P // 4, 16 * 4096, 4096, P // 4, 16 * 4096, 4096, P // 8, 1, None, 0, None, None, 0, out, ld, None, 64, 4096, 4096, 16, 8,
                                     4096, ws, None)

    assert adapt(P, 2 * P, 4096, 0) == ENODEV
    assert adapt(P, P + 2 * 4096, 8192, 0) == ENODEV  # between x's rows
    for x, out, ld in ((P, P, 4096), (P, P + 2, 4096), (P, P + 2 * 4095, 8192), (P + 2 * 63 * 4096 + 2, P, 4096)):
        assert adapt(x, out, ld, in_x - 1) == EINVAL and b"workspace" in lib.skmetal_hip_last_error()
        assert adapt(x, out, ld, in_x) == ENODEV


def test_gradients_share_no_memory_with_what_they_are_made_of(lib):
    def adapt_back(grad=P, x=2 * P, base=None, grad_x=3 * P, ld_base=8):
        return lib.skmetal_hip_adapt_backward(0, grad, 8, x, 8, P // 4, 16, 8, P // 4, 16, 8, P // 8, 1, None, 0, None, P // 2, base, ld_base, grad_x, 8, P // 32, P // 16,
                                              None, 5, 8, 8, 2, 1, 4096, 1 << 30, None)

    assert adapt_back() == ENODEV and adapt_back(base=3 * P) == ENODEV and adapt_back(base=3 * P + 4 * 40) == ENODEV
    for bad in (dict(grad_x=P), dict(grad_x=2 * P + 4 * 39), dict(base=3 * P + 4), dict(base=3 * P, ld_base=16), dict(base=3 * P, ld_base=0)):
        assert adapt_back(**bad) == EINVAL and b"grad_x shares memory" in lib.skmetal_hip_last_error(), bad

    def route_back(grad, ld=8):
        return lib.skmetal_hip_route_backward(0, P, 8, None, 0, 5, 8, 2, 0, P // 2, P // 2, P // 2, P // 2, None, None, grad, ld, None)

    assert route_back(2 * P) == ENODEV and route_back(P) == ENODEV
    for bad in ((P + 4,), (P + 4 * 39,), (P, 9)):
        assert route_back(*bad) == EINVAL and b"grad_logits shares memory" in lib.skmetal_hip_last_error(), bad


@pytest.mark.parametrize("n,d,o,r,a", [(600, 4096, 4096, 16, 2048), (2048, 4096, 4096, 128, 2048), (16_384, 4096, 4096, 64, 2048), (513, 64, 64, 8, 2000),
                                       (100_000, 256, 512, 16, 1000), (16_384, 4096, 4096, 64, 64), (8192, 2048, 2048, 32, 8), (5000, 777, 1001, 5, 1)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_backward_workspace_follows_the_rows(n, d, o, r, a, dtype):
    """Not the adapters, however many: partial sums are those of adapters with more rows than
    a chunk's 64 or more, at most 2 n / 64 of them; beside them the low-rank rows (up to 8
    parts of a sum in fp32, and two sets of three bf16 a rank and up to 256 places more), and a
    few numbers a row and an adapter."""
    from skmetal_amd import _bridge

    rp = -(-r // 16) * 16
    most = 2 * n // 64 * r * (d + o) * 4 + 8 * n * rp * 4 + 12 * r * (n + 256) + 16 * n + 64 * (a + 1) + 8 * (n // 16384 + 1) * (a + 1) + 1024
    size = _bridge._lib.skmetal_hip_adapt_workspace(dtype, n, d, o, r, a, 1)
    assert 0 < size <= most


def test_a_torch_runtime_that_does_not_load_is_named(monkeypatch, tmp_path):
    """KMeans does without it; the operators on torch's tensors say why they cannot run."""
    import importlib.machinery
    import importlib.util
    import io
    import sys

    from skmetal_amd import _bridge

    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "libamdhip64.so").write_text("not a library")
    monkeypatch.delitem(sys.modules, "torch", raising=False)
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: importlib.machinery.ModuleSpec(name, None, origin=str(tmp_path / "__init__.py")))
    monkeypatch.setattr(_bridge, "_torch_runtime_error", None)
    _bridge._share_torch_runtime()
    maps = "7f00-7f01 r-xp 00000000 00:00 0    /a/libamdhip64.so.7\n7f02-7f03 r-xp 00000000 00:00 0    /b/libamdhip64.so\n"
    monkeypatch.setattr("builtins.open", lambda *a, **k: io.StringIO(maps))
    with pytest.raises(RuntimeError, match="two HIP runtimes .*libamdhip64.so: (invalid|file too short)"):
        _bridge.require_torch_runtime()
