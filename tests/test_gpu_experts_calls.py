"""Routing and adapters as callers use them: results in place, inside autograd, on tensors
that other code changes.  Bounds are those of test_gpu_experts."""

from __future__ import annotations

import experts_reference as ref
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import HALF, STEP, TYPES, U, experts, f64, near, part, problem  # noqa: E402, F401 -- a fixture

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,r", [(1, 1024, 8), (64, 4096, 16), (20, 1200, 5), (300, 640, 33), (700, 520, 12)])
def test_out_in_place_of_x(experts, n, d, r, dtype):  # noqa: F811
    """A residual stream in place, where one launch, two and three take the rows: the same
    bits every time, and no column formed from another's result."""
    print("out in x", n, d, r, dtype, flush=True)
    s = problem(n, d, d, r, 5, dtype, n + d)
    opt = dict(gates=s["gates"], scales=s["scales"])
    want, _, mag = ref.adapt(f64(s["x"]), f64(s["down"]), f64(s["up"]), s["ids"].cpu().numpy(), f64(s["x"]), f64(s["gates"]), f64(s["scales"]))
    bound = ((d + r + 16) * U + part(dtype)) * mag + 2 * U * abs(want) + HALF[dtype] * abs(want) + STEP[dtype]
    first = None
    for _ in range(4):
        x = s["x"].clone()
        out = experts.adapt(x, s["down"], s["up"], s["ids"], base=x, out=x, **opt)
        assert out.data_ptr() == x.data_ptr()
        first = out.clone() if first is None else first
        assert torch.equal(out, first)
    near(first, want, bound, "out")
    # rows that lie in x's, one column on: x is read before any of them is written
    wide = torch.zeros(n, d + 8, dtype=TYPES[dtype], device="cuda")
    wide[:, :d] = s["x"]
    out = experts.adapt(wide[:, :d], s["down"], s["up"], s["ids"], base=s["x"], out=wide[:, 1 : d + 1], **opt)
    assert torch.equal(out, first)
    # between x's rows
    both = torch.zeros(n, 2 * d, dtype=TYPES[dtype], device="cuda")
    both[:, :d] = s["x"]
    out = experts.adapt(both[:, :d], s["down"], s["up"], s["ids"], base=s["x"], out=both[:, d:], **opt)
    near(out, want, bound, "out")
    assert torch.equal(both[:, :d], s["x"])


def test_out_partly_in_base_is_refused(experts):  # noqa: F811
    s = problem(9, 32, 24, 4, 3, "bf16", 1)
    wide = torch.zeros(9, 40, dtype=torch.bfloat16, device="cuda")
    for base, out in ((wide[:, :24], wide[:, 1:25]), (wide[:1, :24].expand(9, 24), wide[:, :24]), (wide[1:, :24], wide[:-1, :24])):
        n = out.shape[0]
        with pytest.raises(RuntimeError, match="out shares memory with base"):
            experts.adapt(s["x"][:n], s["down"], s["up"], s["ids"][:n], base=base, out=out)
    experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=wide[:, :12].repeat(1, 2), out=wide[:, 16:])


@pytest.mark.parametrize("normalize", [False, True])
def test_routed_results_changed_in_place(experts, normalize):  # noqa: F811
    """Statistics summed up and a loss weighted in place leave the gradient as it is."""
    g = torch.Generator().manual_seed(1)
    z, dw = torch.randn(300, 24, generator=g).cuda(), torch.randn(300, 3, generator=g).cuda()
    mask = (torch.rand(300, generator=g) < 0.8).cuda()
    plain = experts.route(z, 3, mask=mask, normalize=normalize)
    want = experts.route_backward(z, plain, grad_weights=dw, grad_loss=torch.tensor(0.25, device="cuda"), mask=mask, normalize=normalize)
    z.requires_grad_()
    q = experts.routed(z, 3, mask=mask, normalize=normalize)
    for got, same in zip(q, plain):
        assert torch.equal(got, same) and got.shape == same.shape and got.dtype == same.dtype
    total, loss = (q.weights * dw).sum(), q.loss
    loss.mul_(0.25)
    loss += total
    q.counts.add_(1000)
    q.prob_sums.zero_()
    q.rows.mul_(8)
    loss.backward()
    assert torch.equal(z.grad, want)
    with torch.no_grad():
        q = experts.routed(z, 3, mask=mask, normalize=normalize)
    assert not q.loss.requires_grad and torch.equal(q.counts, plain.counts)


def test_routed_in_a_graph(experts):  # noqa: F811
    """Forward and gradient captured; each replay on new scores, beside eager work."""
    z = torch.randn(700, 40, device="cuda").bfloat16().requires_grad_()
    dw, dl = torch.randn(700, 2, device="cuda"), torch.ones((), device="cuda")

    def work():
        q = experts.routed(z, 2, normalize=True)
        return [*q, *torch.autograd.grad([q.weights, q.loss], [z], [dw, dl])]

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
            z.copy_(torch.randn(700, 40, device="cuda"))
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("e", [24, 200, 600])
def test_route_infinite_score(experts, e, normalize, dtype):  # noqa: F811
    """+inf is a score: the largest, and its row's probabilities are NaN as a softmax's are.
    Which experts a row takes, the places that hold none, masked rows and the other rows
    stay what they are."""
    g = torch.Generator().manual_seed(e)
    z = torch.randn(60, e, generator=g).to(TYPES[dtype])
    z[3, 7] = z[9, 5] = z[9, 2] = z[20, 1] = float("inf")
    z[9, :2] = -float("inf")
    z[9, 6:] = float("nan")  # leaves 2, 3, 4 and 5
    mask = torch.arange(60) != 20
    clean = z.clone()
    clean[3, 7], clean[9, 5], clean[9, 2] = 100.0, 100.0, 100.0
    clean[20] = 0.0
    z, clean, mask = z.cuda(), clean.cuda(), mask.cuda()
    r, c = (experts.route(t, 6, mask=mask, normalize=normalize) for t in (z, clean))
    assert torch.equal(r.experts, c.experts) and torch.equal(r.counts, c.counts) and torch.equal(r.rows, c.rows)
    assert r.experts[9].tolist()[:2] == [2, 5] and r.experts[9].tolist()[4:] == [-1, -1]
    rest = torch.ones(60, dtype=torch.bool)
    rest[[3, 9]] = False
    assert torch.equal(r.weights[rest], c.weights[rest])
    assert r.weights[3].isnan().all() and r.weights[9, :4].isnan().all() and (r.weights[9, 4:] == 0).all()
    assert r.prob_sums.isnan().any() and r.loss.isnan()
    dw, dl = torch.randn(60, 6, generator=g).cuda(), torch.ones((), device="cuda")
    a, b = (experts.route_backward(t, q, grad_weights=dw, grad_loss=dl, mask=mask, normalize=normalize) for t, q in ((z, r), (clean, c)))
    assert torch.equal(a[rest], b[rest]) and a[3].isnan().any() and (a[20] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,e,k", [(70, 40, 3), (30_001, 200, 4)])
def test_gradient_of_the_scores_in_their_place(experts, n, e, k, dtype):  # noqa: F811
    """The C entry's grad_logits over logits, from one group of rows a wave and from several."""
    g = torch.Generator().manual_seed(n)
    z = torch.randn(n, e, generator=g).to(TYPES[dtype]).cuda()
    dw, dl = torch.randn(n, k, generator=g).cuda(), torch.ones((), device="cuda")
    r = experts.route(z, k)
    want = experts.route_backward(z, r, grad_weights=dw, grad_loss=dl)
    code = experts._lib().skmetal_hip_route_backward(experts._CODE[z.dtype], z.data_ptr(), e, None, 0, n, e, k, 0, r.weights.data_ptr(), r.experts.data_ptr(), r.counts.data_ptr(),
                                                     r.rows.data_ptr(), dw.data_ptr(), dl.data_ptr(), z.data_ptr(), e, experts._stream(z.device))
    assert code == 0 and torch.equal(z, want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [20, 150, 700])
def test_gradient_of_the_rows_in_place_of_its_base(experts, n, dtype):  # noqa: F811
    """The C entry's grad_x over its base."""
    d, o, r, a = 1100, 96, 20, 4
    s = problem(n, d, o, r, a, dtype, n)
    _, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], return_low=True)
    want = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, base=s["grad_base"])
    place, down, up = s["grad_base"].clone(), torch.empty_like(s["down"]), torch.empty_like(s["up"])
    code, stream = experts._CODE[TYPES[dtype]], experts._stream(place.device)
    size = experts._adapt_workspace(code, n, d, o, r, a, 1)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    at = place.data_ptr()
    done = experts._lib().skmetal_hip_adapt_backward(code, s["grad"].data_ptr(), o, s["x"].data_ptr(), d, s["down"].data_ptr(), r * d, d, s["up"].data_ptr(), r * o, o, s["ids"].data_ptr(),
                                                     1, None, 0, None, low.data_ptr(), at, d, at, d, down.data_ptr(), up.data_ptr(), None, n, d, o, r, a, ws.data_ptr(), size, stream)
    assert done == 0
    assert torch.equal(place, want.x) and torch.equal(down, want.down) and torch.equal(up, want.up)
