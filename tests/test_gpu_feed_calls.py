"""Feed-forward, dropout and log probabilities as a program uses them: one after the other as a model's step,
served row by row, on other streams, and captured into graphs."""

from __future__ import annotations

import feed_reference as ref
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import U, experts, f64  # noqa: E402, F401 -- a fixture
from test_gpu_feed import problem  # noqa: E402

pytestmark = pytest.mark.gpu


def model(n, d, f, v, e, r, seed):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).cuda()

    return dict(x=normal(n, d), centres=normal(e, d, std=0.5), gate=normal(e, f, d, std=d**-0.5), up=normal(e, f, d, std=d**-0.5), down=normal(e, d, f, std=f**-0.5),
                a=normal(e, r, d, std=d**-0.5), b=normal(e, r, v, std=0.1), head=normal(v, d, std=d**-0.5)), torch.randint(0, v, (n,), generator=g).int().cuda()


def step(experts, m, targets, key):  # noqa: F811
    """A router's experts, dropout beside the residual stream, a head with an adapter per first choice, the loss."""
    logits = m["x"] @ m["centres"].T.contiguous()
    q = experts.routed(logits, 2, normalize=True)
    h = experts.fed(m["x"], m["gate"], m["up"], m["down"], q.experts, weights=q.weights)
    y = experts.dropped(h, 0.25, key, site=3, base=m["x"])
    z = experts.adapted(y, m["a"], m["b"], q.experts[:, 0], base=y @ m["head"].T)
    t = experts.rated(z, targets, top_k=3)
    return -t.log_probs.mean() - 0.01 * t.entropy.mean() + 0.1 * q.loss, q, t


def test_a_step_of_a_model(experts):  # noqa: F811
    """Against torch's autograd in 64 bits, with the router's choice and the mask as they came: chains of fp32
    sums of under 700 terms, 2^-24 each, 3e-5 of the norm."""
    n, d, f, v, e = 130, 48, 72, 90, 6
    m, targets = model(n, d, f, v, e, 4, 1)
    key = torch.tensor([11, 5], device="cuda")
    for t in m.values():
        t.requires_grad_()
    loss, q, rating = step(experts, m, targets, key)
    got = torch.autograd.grad(loss, list(m.values()))
    w = {k: t.detach().double().requires_grad_() for k, t in m.items()}
    keep = torch.from_numpy((ref.words(n * d, 11, 5, 3) >= 2**30).reshape(n, d)).cuda()
    p = torch.softmax(w["x"] @ w["centres"].T, 1)
    c = q.experts.long()
    pw = p.gather(1, c)
    pw = pw / pw.sum(1, keepdim=True)
    h = 0
    for j in range(2):
        g = (w["gate"][c[:, j]] * w["x"][:, None, :]).sum(2)
        u = (w["up"][c[:, j]] * w["x"][:, None, :]).sum(2)
        h = h + pw[:, j, None] * (w["down"][c[:, j]] * (torch.nn.functional.silu(g) * u)[:, None, :]).sum(2)
    y = w["x"] + torch.where(keep, h / 0.75, 0.0)
    z = y @ w["head"].T + (w["b"][c[:, 0]] * (w["a"][c[:, 0]] * y[:, None, :]).sum(2)[:, :, None]).sum(1)
    lp = torch.log_softmax(z, 1)
    entropy = -(lp.exp() * lp).sum(1)
    counts = torch.bincount(c.flatten(), minlength=e).double()
    want_loss = -lp.gather(1, targets.long()[:, None]).mean() - 0.01 * entropy.mean() + 0.1 * e / (2 * n * n) * (counts * p.sum(0)).sum()
    want = torch.autograd.grad(want_loss, list(w.values()))
    assert abs(loss.item() - want_loss.item()) < 1e-5 * abs(want_loss.item())
    assert (rating.top[:, 0] == z.argmax(1)).float().mean() > 0.98  # near ties aside
    for name, a, b in zip(m, got, want):
        assert float((a.double() - b).norm()) < 3e-5 * float(b.norm()), name


def test_served_rows_are_the_batch(experts):  # noqa: F811
    """One row, a few and many take other launches; the results are the batch's, but for the order of fp32 sums
    (bf16: 128 terms of products, then one rounding each of h and out, and h's passed on: 4 2^-8 of the largest)."""
    s = problem(300, 128, 128, 128, 6, 2, "bf16", 4)
    m = s["gate"], s["up"], s["down"]
    want = experts.feed(s["x"], *m, s["chosen"], weights=s["weights"], base=s["base"]).float()
    for n in (1, 2, 7, 9, 33):
        got = experts.feed(s["x"][:n], *m, s["chosen"][:n], weights=s["weights"][:n], base=s["base"][:n]).float()
        assert float((got - want[:n]).abs().max()) <= 4 * 2.0**-8 * float(want.abs().max())
    z, t = torch.randn(40, 5000, device="cuda"), torch.arange(40, device="cuda").int()
    want = experts.rate(z, t, top_k=4)
    for i in (0, 17, 39):
        one = experts.rate(z[i : i + 1], t[i : i + 1], top_k=4)
        assert torch.equal(one.top[0], want.top[i]) and float((one.log_probs - want.log_probs[i]).abs()) < 64 * U * 20
    key = torch.tensor([1, 2], device="cuda")
    assert torch.equal(experts.drop(z, 0.5, key)[0], experts.drop(z[:1], 0.5, key)[0])


@pytest.mark.parametrize("n", [3, 400])
def test_another_stream_and_a_graph(experts, n):  # noqa: F811
    """Few slots and many; every replay on new rows, choices and a new step of the mask, beside eager work."""
    print("graph", n, flush=True)
    s = problem(n, 96, 128, 96, 5, 2, "bf16", 3)
    m = s["gate"], s["up"], s["down"]
    key = torch.tensor([77, 0], device="cuda")
    z, t = torch.randn(n, 9000, device="cuda"), torch.randint(0, 9000, (n,), device="cuda").int()
    ones = torch.ones(n, device="cuda")

    def work():
        out, pre = experts.feed(s["x"], *m, s["chosen"], weights=s["weights"], base=s["base"], return_pre=True)
        g = experts.feed_backward(s["grad"], s["x"], *m, s["chosen"], pre, weights=s["weights"])
        y = experts.drop(out, 0.25, key, site=9, base=s["x"])
        r = experts.rate(z, t, top_k=5)
        return [out, pre, *g, y, *r, experts.rate_backward(z, t, r, grad_log_probs=ones, grad_entropy=ones)]

    want = work()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = work()
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
        key[1] += 1
    masks = []
    for i in range(4):
        s["x"].copy_(torch.randn(n, 96, device="cuda"))
        s["chosen"].copy_(torch.randint(-1, 6, (n, 2), device="cuda"))
        z.copy_(torch.randn(n, 9000, device="cuda"))
        before = int(key[1])
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        assert int(key[1]) == before + 1
        for a, b in zip(held, want):
            assert torch.equal(a, b), i
        masks.append((held[7] == s["x"]).clone())
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


def test_gradients_in_a_graph(experts):  # noqa: F811
    """A whole step captured, forward and gradients; each replay on new rows and another mask."""
    m, targets = model(200, 64, 96, 120, 5, 4, 2)
    for t in m.values():
        t.requires_grad_()
    key = torch.tensor([3, 0], device="cuda")

    def work():
        loss, _, _ = step(experts, m, targets, key)
        return [loss.detach(), *torch.autograd.grad(loss, list(m.values()))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(4):
        with torch.no_grad():
            m["x"].copy_(torch.randn(200, 64, device="cuda"))
            key[1] = 10 + i
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):  # torch's own products may split their sums otherwise in a graph: 2e-5 of the norm
            assert float((a - b).norm()) <= 2e-5 * float(b.norm()), i


def test_two_graphs_at_once(experts):  # noqa: F811
    """Two graphs with workspaces of their own, replayed on two streams together."""
    problems = [problem(500, 64, 96, 64, 4, 2, "bf16", i) for i in (1, 2)]
    graphs, held = [], []

    def work(s):
        out, pre = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], return_pre=True)
        return [out, *experts.feed_backward(s["grad"], s["x"], s["gate"], s["up"], s["down"], s["chosen"], pre, weights=s["weights"])]

    want = [work(s) for s in problems]
    for s in problems:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(work(s))
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(5):
        for st, gr in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            for a, b in zip(h, w):
                assert torch.equal(a, b)


def test_rows_behind_the_last_are_left_alone(experts):  # noqa: F811
    """out within larger storage: rows and columns around it stay what they were."""
    for n, k in ((2, 2), (150, 1), (150, 2)):
        s = problem(n, 64, 72, 48, 3, k, "bf16", 8)
        room = torch.full((n + 3, 60), 5.0, device="cuda", dtype=torch.bfloat16)
        want = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"])
        experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], out=room[1 : n + 1, 4:52])
        assert torch.equal(room[1 : n + 1, 4:52], want)
        room[1 : n + 1, 4:52] = 5.0
        assert (room == 5).all()
        experts.drop(s["x"][:, :48], 0.5, torch.tensor([1, 1], device="cuda"), out=room[1 : n + 1, 4:52])
        room[1 : n + 1, 4:52] = 5.0
        assert (room == 5).all()


def test_workspace_is_not_kept(experts):  # noqa: F811
    """Nothing of one call is left for the next: the same call after others, with scratch full of NaN, gives the same bits."""
    s = problem(260, 96, 136, 64, 4, 2, "bf16", 6)
    m = s["gate"], s["up"], s["down"]

    def work():
        out, pre = experts.feed(s["x"], *m, s["chosen"], weights=s["weights"], return_pre=True)
        g = experts.feed_backward(s["grad"], s["x"], *m, s["chosen"], pre, weights=s["weights"])
        z = experts.rate(s["x"].float().repeat(1, 100), s["chosen"][:, 0].contiguous(), top_k=16)
        return [out, pre, *g, *z]

    want = work()
    for _ in range(3):
        junk = [torch.full((1 << i,), float("nan"), device="cuda") for i in range(8, 24)]
        torch.cuda.synchronize()
        del junk  # goes back to the allocator, and to the calls as scratch
        for a, b in zip(work(), want):
            assert torch.equal(a, b)


def test_sixteen_choices_and_many_experts(experts):  # noqa: F811
    """The widest choice, with every expert of a row the same, and more experts than rows."""
    s = problem(40, 24, 40, 16, 2048, 16, "fp32", 2)
    s["chosen"] = torch.randint(0, 2048, (40, 16), generator=torch.Generator().manual_seed(1)).int().cuda()
    s["chosen"][3] = 77
    m = s["gate"], s["up"], s["down"]
    out, pre = experts.feed(s["x"], *m, s["chosen"], weights=s["weights"], return_pre=True)
    g = experts.feed_backward(s["grad"], s["x"], *m, s["chosen"], pre, weights=s["weights"])
    want = ref.feed(f64(s["x"]), *(f64(t) for t in m), s["chosen"].cpu().numpy(), f64(s["weights"]), grad=f64(s["grad"]))
    for got, (v, bound) in ((out, want["out"]), (g.x, want["x"]), (g.gate, want["gate"]), (g.down, want["down"]), (g.weights, want["weights"])):
        assert (np.abs(f64(got) - v) <= bound).all()
