"""What the operators of skmetal_amd.experts hand to the library for batches of no rows, without a GPU.  Of an empty
matrix no stride says anything: that of a broadcast gradient is 0, and ``contiguous`` leaves it."""

from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def calls(monkeypatch):
    """The entry points that were reached."""
    from skmetal_amd import experts

    made = []

    def entry(name):
        return lambda *args: made.append(name) or 0

    names = ("route", "route_backward", "adapt", "adapt_backward", "feed", "feed_backward", "drop", "rate", "rate_backward")
    monkeypatch.setattr(experts, "_lib", lambda: types.SimpleNamespace(**{f"skmetal_hip_{n}": entry(n) for n in names}))
    monkeypatch.setattr(experts, "_first", lambda t, name: (experts._CODE[t.dtype], t.device))
    monkeypatch.setattr(experts, "_stream", lambda device: None)
    for size in ("route", "adapt", "feed", "rate"):
        monkeypatch.setattr(experts, f"_{size}_workspace", lambda *sizes: 0)
    return made


def test_broadcast_gradient_of_no_rows(calls):
    from skmetal_amd import experts

    x = torch.zeros(0, 16, requires_grad=True)
    key, chosen = torch.zeros(2, dtype=torch.int64), torch.zeros(0, 2, dtype=torch.int32)
    experts.fed(x, torch.zeros(3, 8, 16), torch.zeros(3, 8, 16), torch.zeros(3, 16, 8), chosen).sum().backward()
    experts.dropped(x, 0.1, key).sum().backward()
    experts.adapted(x, torch.zeros(3, 4, 16), torch.zeros(3, 4, 16), chosen[:, 0]).sum().backward()
    r = experts.rated(x, chosen[:, 0])
    (r.log_probs.sum() + r.entropy.sum()).backward()
    q = experts.routed(x, 2)
    (q.weights.sum() + q.loss).backward()
    assert calls == ["feed", "feed_backward", "drop", "drop", "adapt", "adapt_backward", "rate", "rate_backward", "route", "route_backward"]
    assert x.grad.shape == (0, 16)


def test_no_rows_with_strides_of_their_own(calls):
    """A transposed or expanded tensor without rows."""
    from skmetal_amd import experts

    t, key, chosen = torch.zeros(0, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(0, 1, dtype=torch.int32)
    m = torch.zeros(2, 8, 16), torch.zeros(2, 8, 16), torch.zeros(2, 16, 8)
    for x in (torch.zeros(16, 4).T[:0], torch.zeros(1, 1).expand(1, 16)[:0]):
        assert x.shape == (0, 16) and x.stride(1) != 1
        experts.feed(x, *m, chosen, base=x)
        experts.drop(x, 0.1, key, base=x)
        experts.rate(x, t)
        experts.route(x, 2)
        experts.adapt(x, torch.zeros(2, 4, 16), torch.zeros(2, 4, 16), t, base=x)
    assert calls == ["feed", "drop", "rate", "route", "adapt"] * 2


def test_rows_apart_are_still_refused(calls):
    from skmetal_amd import experts

    x, t, key = torch.zeros(16, 5).T, torch.zeros(5, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: experts.drop(x, 0.1, key), lambda: experts.rate(x, t), lambda: experts.route(x, 2), lambda: experts.adapt(x, torch.zeros(2, 4, 16), torch.zeros(2, 4, 16), t)):
        with pytest.raises(ValueError, match="side by side"):
            call()
    assert not calls
