"""Feed-forward calls at the edges of what their documentation allows, on the GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import TYPES, experts  # noqa: E402, F401 -- a fixture
from test_gpu_feed import check, problem  # noqa: E402

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


@pytest.mark.parametrize("n", [16, 300])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activation_keeps_its_bits(experts, act, n):  # noqa: F811
    """One product a sum, so that out is the activation and grad_gate its derivative, in fp32, each relative to itself.

    In u = 2^-24.  gelu: x and its constant 1.5, t = rcp 3, t P(t) follows t at most in proportion, P's sum 3 and its fit 2.5, the
    exponential 5 (exp2 2, three roundings), three products 3, the last 1: 20.  silu: the exponential 5, a sum 1, rcp 2, the last 1: 9, so 12.
    Derivatives: as much of c + |g phi| or t (1 + |g|), with two roundings.  Below 2^-126 nothing is relative."""
    gen = torch.Generator().manual_seed(n)
    g = (torch.rand(n, n, generator=gen) * 21.2 - 13.2) if act == "gelu" else torch.rand(n, n, generator=gen) * 107.0 - 87.0
    one = torch.eye(n, device="cuda")
    out, pre = experts.feed(one, g.T.contiguous().cuda()[None], torch.ones(1, n, n, device="cuda"), one[None], act=act, return_pre=True)
    assert torch.equal(pre[:, 0, 0].cpu(), g) and (pre[:, 0, 1] == 1).all()
    grads = experts.feed_backward(torch.ones(n, n, device="cuda"), one, g.T.contiguous().cuda()[None], torch.ones(1, n, n, device="cuda"), one[None], None, pre, act=act)
    z, u = g.double(), 2.0**-24
    if act == "gelu":
        c, slope = 0.5 * torch.special.erfc(-z / 2**0.5), z * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
        want, derivative, size, bound = z * c, c + slope, c + slope.abs(), 20 * u
    else:
        c = torch.sigmoid(z)
        want, derivative, size, bound = z * c, c * (1 + z * torch.sigmoid(-z)), c * (1 + z.abs()), 12 * u
    least = 16 * 2.0**-126
    off = (out.double().cpu() - want).abs() - least
    assert (off <= bound * want.abs()).all(), (off / want.abs()).max() / u
    off = (grads.gate[0].T.double().cpu() - derivative).abs() - least
    assert (off <= (bound + 2 * u) * size).all(), (off / size).max() / u


@pytest.mark.parametrize("n,d,f,a,k,dtype", [(12, 4096, 2048, 1, 1, "bf16"), (24, 2048, 1024, 2, 2, "fp16"), (24, 4096, 2048, 1, 1, "fp32"), (60, 2047, 1023, 2, 1, "bf16"), (8, 4096, 2048, 4, 2, "fp32")])
def test_few_slots_that_share_experts(experts, n, d, f, a, k, dtype):  # noqa: F811
    """Up to 64 slots by tiles, which read an expert's matrices once, and the first rows by themselves, slot by slot."""
    print("shared", n, d, f, a, k, dtype, flush=True)
    s = problem(n, d, f, d, a, k, dtype, n)
    check(experts, s, dtype, dense=a == 1, backward=False)
    check(experts, {name: t if name in ("gate", "up", "down") else t[:2] for name, t in s.items()}, dtype, dense=a == 1, backward=False)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,f", [(9, 64, 48), (500, 128, 320), (300, 65, 33), (2600, 64, 4104)])
def test_one_block_with_and_without_a_choice(experts, n, d, f, dtype):  # noqa: F811
    """chosen None is every row's choice of the one expert: the same places in the same tiles, bit for bit in both directions."""
    print("one block", n, d, f, dtype, flush=True)
    s = problem(n, d, f, d, 1, 1, dtype, n)
    m, zeros = (s["gate"], s["up"], s["down"]), torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    results = []
    for chosen in (None, zeros):
        out, pre = experts.feed(s["x"], *m, chosen, weights=s["weights"], base=s["base"], return_pre=True)
        results.append([out, pre, *experts.feed_backward(s["grad"], s["x"], *m, chosen, pre, weights=s["weights"], base=s["grad_base"])])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [8, 300])
def test_fp16_range(experts, n):  # noqa: F811
    """A weighted hidden value past 65,504 is infinite, in its row alone; the weight comes first; gradients keep fp16's smallest
    step (which the reference's bounds count)."""
    s = problem(n, 64, 96, 64, 3, 1, "fp16", 4)
    s["chosen"][:, 0] = torch.arange(n, device="cuda").int() % 3
    m = s["gate"], s["up"], s["down"]
    plain = experts.feed(s["x"], *m, s["chosen"], base=s["base"])
    s["x"][5] *= 400
    rest = torch.arange(n, device="cuda") != 5
    out = experts.feed(s["x"], *m, s["chosen"], base=s["base"])
    assert not torch.isfinite(out[5]).all() and torch.equal(out[rest], plain[rest])
    s["weights"][5] = 2.0**-10
    s["grad"] *= 2.0**-12
    assert torch.isfinite(check(experts, s, "fp16")).all()


@pytest.mark.parametrize("n", [3, 70])
def test_places_past_32_bits(experts, n):  # noqa: F811
    """Rows and experts that lie more than 2^31 and 2^32 elements apart, in one allocation that is read only where they are."""
    print("far", n, flush=True)
    a, d, f, far = 3, 64, 40, 2**31 + 64
    s = problem(n, d, f, d, a, 2, "bf16", 5)
    room = torch.empty(3 * far, dtype=torch.bfloat16, device="cuda")
    step = 2 * far // n // 64 * 64
    place, views = 0, {}
    for name in ("x", "base", "grad", "grad_base"):
        views[name] = room.as_strided(s[name].shape, (step, 1), place)
        place += d
    for name in ("gate", "up", "down"):
        views[name] = room.as_strided(s[name].shape, (far, s[name].shape[2], 1), place)
        place += s[name][0].numel()
    assert (n - 1) * step > 2**31 and place < step
    for name, view in views.items():
        view.copy_(s[name])
    want = check(experts, s, "bf16")
    assert torch.equal(check(experts, {**s, **views}, "bf16"), want)
    got = experts.feed(views["x"], views["gate"], views["up"], views["down"], s["chosen"], weights=s["weights"], base=views["base"], out=views["base"])
    assert torch.equal(got, want)
    z, t = room.as_strided((n, 3000), (step, 1), place), torch.arange(n, device="cuda").int()
    z.copy_(torch.randn(n, 3000, device="cuda"))
    near, far_away = (experts.rate(v, t, top_k=3) for v in (z.contiguous(), z))
    assert all(torch.equal(p, q) for p, q in zip(near, far_away))
    assert torch.equal(*(experts.rate_backward(v, t, near, grad_log_probs=torch.ones(n, device="cuda")) for v in (z, z.contiguous())))
