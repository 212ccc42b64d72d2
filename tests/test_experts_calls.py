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
