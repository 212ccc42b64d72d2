"""Gated feed-forward blocks of experts on the GPU against their formulas in 64 bits; the bounds
are the reference's (feed_reference)."""

from __future__ import annotations

import math

import feed_reference as ref
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import TYPES, experts, f64, near  # noqa: E402, F401 -- a fixture

pytestmark = pytest.mark.gpu


def problem(n, d, f, o, a, k, dtype, seed, law="some"):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(t).cuda()

    chosen = torch.randint(-1, a + 1, (n, k), generator=g)  # -1 and a: none; an expert twice in a row too
    if law == "one":
        chosen = torch.full((n, k), a - 1)
    elif law == "none":
        chosen = torch.full((n, k), -1)
    elif law == "wild":
        chosen[torch.rand(n, k, generator=g) < 0.3] = -(2**31)
        chosen[torch.rand(n, k, generator=g) < 0.3] = 2**31 - 1
    return dict(x=normal(n, d), gate=normal(a, f, d, std=1 / math.sqrt(d)), up=normal(a, f, d, std=1 / math.sqrt(d)), down=normal(a, o, f, std=1 / math.sqrt(f)),
                chosen=chosen.int().cuda(), weights=torch.rand(n, k, generator=g).cuda(), base=normal(n, o), grad=normal(n, o), grad_base=normal(n, d))


def check(experts, s, dtype, act="silu", weights=True, base=True, dense=False, backward=True):  # noqa: F811
    x, m, chosen = s["x"], (s["gate"], s["up"], s["down"]), s["chosen"]
    n = x.shape[0]
    opt = dict(weights=s["weights"] if weights else None, act=act)
    given = None if dense else chosen
    out, pre = experts.feed(x, *m, given, base=s["base"] if base else None, return_pre=True, **opt)
    bare = experts.feed(x, *m, given, base=s["base"] if base else None, **opt)
    assert out.dtype == x.dtype and torch.equal(out, bare)
    I = np.zeros((n, 1), np.int64) if dense else chosen.cpu().numpy()
    want = ref.feed(f64(x), *(f64(v) for v in m), I, f64(s["weights"]) if weights else None, f64(s["base"]) if base else None, act, dtype,
                    f64(s["grad"]) if backward else None, f64(s["grad_base"]) if base else None)
    near(pre, *want["pre"], "pre")
    near(out, *want["out"], "out")
    if not backward:
        return out
    args = (s["grad"], x, *m, given, pre)
    g = experts.feed_backward(*args, base=s["grad_base"] if base else None, **opt)
    again = experts.feed_backward(*args, base=s["grad_base"] if base else None, **opt)
    for name in ("x", "gate", "up", "down", "weights"):
        got = getattr(g, name)
        if name == "weights" and not weights:
            assert got is None
            continue
        assert torch.equal(got, getattr(again, name)), name
        near(got, *want[name], f"grad_{name}")
    rows = experts.feed_backward(*args, base=s["grad_base"] if base else None, matrices=False, **opt)
    assert torch.equal(rows.x, g.x) and rows.gate is rows.up is rows.down is None and (not weights or torch.equal(rows.weights, g.weights))
    matrices = experts.feed_backward(*args, rows=False, **opt)
    assert matrices.x is None and all(torch.equal(getattr(matrices, v), getattr(g, v)) for v in ("gate", "up", "down"))
    return out


# n, d, f, o, a, k: one row, odd widths, tiles that end inside an expert, one term, many experts
SIZES = [(1, 64, 64, 64, 1, 1), (1, 256, 128, 256, 8, 2), (5, 33, 17, 41, 3, 2), (3, 1, 1, 1, 1, 1), (70, 72, 40, 24, 4, 3), (300, 96, 160, 96, 5, 2), (37, 8, 200, 16, 2, 16),
         (130, 130, 65, 258, 3, 1), (64, 520, 264, 136, 16, 4), (1, 1000, 24, 40, 70, 5), (20, 40, 48, 56, 300, 2)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,f,o,a,k", SIZES)
def test_feed(experts, n, d, f, o, a, k, dtype):  # noqa: F811
    print("feed", n, d, f, o, a, k, dtype, flush=True)
    check(experts, problem(n, d, f, o, a, k, dtype, n + d), dtype, act=("silu", "gelu", "relu")[(n + k) % 3])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,f,o,a,k", [(1500, 128, 192, 128, 3, 2), (700, 264, 72, 40, 2, 1), (4000, 64, 512, 64, 2, 3), (2000, 777, 40, 33, 2, 1), (17000, 16, 24, 8, 9, 1)])
def test_feed_many_rows(experts, n, d, f, o, a, k, dtype):  # noqa: F811
    """Several tiles an expert, sums over the rows in parts, several segments of the sort."""
    print("feed", n, d, f, o, a, k, dtype, flush=True)
    check(experts, problem(n, d, f, o, a, k, dtype, n + d), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_feed_largest_tiles(experts, dtype):  # noqa: F811
    """Enough rows and columns for the largest tiles, whose last ones are cut on both sides."""
    print("feed largest", dtype, flush=True)
    check(experts, problem(4200, 72, 4104, 40, 3, 1, dtype, 5), dtype)
    check(experts, problem(2100, 136, 4104, 72, 2, 2, dtype, 6), dtype, act="gelu")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("law", ["one", "none", "wild"])
@pytest.mark.parametrize("n,d,f,o,a,k", [(9, 72, 48, 16, 4, 2), (300, 64, 65, 33, 3, 1), (400, 40, 24, 32, 20, 3)])
def test_feed_choices(experts, n, d, f, o, a, k, law, dtype):  # noqa: F811
    print("feed", law, n, d, f, o, a, k, dtype, flush=True)
    check(experts, problem(n, d, f, o, a, k, dtype, n + d, law), dtype)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("base", [False, True])
def test_feed_options(experts, act, weights, base):  # noqa: F811
    for dtype, n, k in (("bf16", 5, 1), ("fp32", 200, 2), ("fp16", 300, 1)):
        check(experts, problem(n, 64, 96, 80, 4, k, dtype, 21), dtype, act, weights, base)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,f,o", [(1, 64, 128, 64), (17, 65, 33, 40), (500, 128, 320, 96), (2, 1032, 40, 8)])
def test_feed_one_block_for_all_rows(experts, n, d, f, o, dtype):  # noqa: F811
    print("dense", n, d, f, o, dtype, flush=True)
    s = problem(n, d, f, o, 1, 1, dtype, n)
    out = check(experts, s, dtype, dense=True)
    s["chosen"][:] = 0
    assert torch.equal(out, experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], base=s["base"])) or n > 1


def test_feed_strides_and_places(experts):  # noqa: F811
    """Rows apart, rows off any 16-byte line, matrices cut out of larger ones or halves of
    one, an expanded row, and out in base's place."""
    for dtype in TYPES:
        for n in (9, 333):
            s = problem(n, 101, 60, 90, 3, 2, dtype, 6)
            wide = problem(n, 160, 200, 128, 5, 2, dtype, 7)
            s["x"], s["base"] = wide["x"][:, 3:104], wide["base"][:, 5:95]
            s["grad"], s["grad_base"] = wide["grad"][:, 1:91], wide["grad_base"][:, 7:108]
            s["gate"], s["up"] = wide["gate"][1:4, 2:62, 9:110], wide["gate"][1:4, 62:122, 9:110]
            s["down"] = wide["down"][2:5, 2:92, 11:71]
            want = check(experts, s, dtype)
            place = torch.full((n, 128), 3.0, dtype=TYPES[dtype], device="cuda")
            place[:, 5:95] = s["base"]
            got = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], base=place[:, 5:95], out=place[:, 5:95])
            assert got.data_ptr() == place[:, 5:95].data_ptr() and torch.equal(got, want)
            assert (place[:, :5] == 3).all() and (place[:, 95:] == 3).all()
    s = problem(50, 64, 48, 64, 3, 2, "bf16", 6)
    s["x"], s["base"] = s["x"][:1].expand(50, 64), s["base"][:1].expand(50, 64)
    check(experts, s, "bf16")


def test_feed_residual_in_place(experts):  # noqa: F811
    """x, base and out one tensor: rows are read before any is written."""
    for n, k in ((1, 1), (40, 2), (600, 1)):
        s = problem(n, 64, 96, 64, 4, k, "bf16", 3)
        want = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], base=s["x"])
        x = s["x"].clone()
        assert torch.equal(experts.feed(x, s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"], base=x, out=x), want)


def test_feed_rows_without_an_expert_touch_nothing(experts):  # noqa: F811
    """NaN and infinity in rows without an expert, and in experts that no row has, stay where they are."""
    for n, k in ((11, 2), (600, 1), (400, 2)):
        for d in (64, 65):
            s = problem(n, d, 48, 40, 4, k, "bf16", 13)
            s["chosen"][s["chosen"] == 2] = 0
            none = ((s["chosen"] < 0) | (s["chosen"] >= 4)).all(1)
            s["chosen"][: n // 3] = -1
            none[: n // 3] = True
            for name in ("x", "weights", "grad"):
                s[name][none] = math.nan
            s["gate"][2], s["up"][2], s["down"][2] = math.inf, math.nan, math.nan
            opt = dict(weights=s["weights"])
            m = s["gate"], s["up"], s["down"]
            out, pre = experts.feed(s["x"], *m, s["chosen"], base=s["base"], return_pre=True, **opt)
            assert torch.isfinite(out).all() and torch.equal(out[none], s["base"][none]) and (pre[none] == 0).all()
            g = experts.feed_backward(s["grad"], s["x"], *m, s["chosen"], pre, base=s["grad_base"], **opt)
            assert all(torch.isfinite(t).all() for t in g) and torch.equal(g.x[none], s["grad_base"][none]) and (g.weights[none] == 0).all()
            assert (g.gate[2] == 0).all() and (g.up[2] == 0).all() and (g.down[2] == 0).all()


def test_feed_an_infinity_reaches_its_row_alone(experts):  # noqa: F811
    for n in (8, 500):
        s = problem(n, 64, 48, 40, 4, 1, "bf16", 14)
        s["chosen"][:, 0] = torch.arange(n, device="cuda").int() % 4
        plain = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"])
        s["x"][5, 3] = math.inf
        out = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"])
        rest = torch.arange(n, device="cuda") != 5
        assert not torch.isfinite(out[5]).all() and torch.equal(out[rest], plain[rest])


def test_feed_nothing_to_do(experts):  # noqa: F811
    s = problem(0, 16, 24, 32, 3, 2, "bf16", 1)
    out, pre = experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], return_pre=True)
    assert out.shape == (0, 32) and pre.shape == (0, 2, 2, 24)
    g = experts.feed_backward(s["grad"], s["x"], s["gate"], s["up"], s["down"], s["chosen"], pre, weights=s["weights"])
    assert g.x.shape == (0, 16) and g.weights.shape == (0, 2) and all((t == 0).all() and t.shape == s[v].shape for v, t in (("gate", g.gate), ("up", g.up), ("down", g.down)))
    s = problem(0, 16, 24, 32, 1, 1, "fp32", 1)
    _, pre = experts.feed(s["x"], s["gate"], s["up"], s["down"], return_pre=True)
    assert (experts.feed_backward(s["grad"], s["x"], s["gate"], s["up"], s["down"], None, pre).down == 0).all()


def test_feed_extreme_activations(experts):  # noqa: F811
    """g far on both sides: act's limits, no NaN from an overflowing exponential."""
    s = problem(6, 8, 8, 8, 1, 1, "fp32", 2)
    s["x"][:] = torch.eye(8, device="cuda")[:6]
    s["gate"][0] = torch.tensor([-1e30, -200.0, -95.0, 0.0, 95.0, 200.0, 1e18, -0.0], device="cuda")[:, None].expand(8, 8)
    s["chosen"][:] = 0
    for act in ("silu", "gelu", "relu"):
        check(experts, s, "fp32", act)


def test_fed_gradients(experts):  # noqa: F811
    """Autograd's own chain in 64 bits: fp32 sums of under 300 terms at 2^-24 each, 2e-5 of the norm."""
    torch.manual_seed(0)
    n, d, f, o, a, k = 90, 32, 48, 24, 5, 2
    x = torch.randn(n, d, device="cuda", requires_grad=True)
    gate, up = (torch.randn(a, f, d, device="cuda", requires_grad=True) for _ in range(2))
    down, base = torch.randn(a, o, f, device="cuda", requires_grad=True), torch.randn(n, o, device="cuda", requires_grad=True)
    chosen = torch.randint(-1, a, (n, k), device="cuda").int()
    w = torch.rand(n, k, device="cuda", requires_grad=True)
    v = [x, gate, up, down, w, base]
    got = torch.autograd.grad(experts.fed(x, gate, up, down, chosen, weights=w, base=base, act="gelu").square().sum(), v)
    x2, g2, u2, d2, w2, b2 = (t.detach().double().requires_grad_() for t in v)
    y = b2
    for j in range(k):
        q = chosen[:, j].long().clamp(min=0)
        h = torch.nn.functional.gelu((g2[q] * x2[:, None, :]).sum(2)) * (u2[q] * x2[:, None, :]).sum(2)
        y = y + torch.where(chosen[:, j, None] >= 0, w2[:, j, None] * (d2[q] * h[:, None, :]).sum(2), 0.0)
    want = torch.autograd.grad(y.square().sum(), [x2, g2, u2, d2, w2, b2])
    for p, q in zip(got, want):
        assert float((p.double() - q).norm()) < 2e-5 * float(q.norm())


@pytest.mark.parametrize("frozen", [(), ("gate", "up", "down"), ("x",), ("x", "weights"), ("x", "gate", "up", "down")])
def test_fed_frozen_parts(experts, frozen):  # noqa: F811
    s = problem(60, 32, 24, 32, 3, 2, "fp32", 9)
    names = ("x", "gate", "up", "down", "weights", "base")
    every = {v: s[v].clone().requires_grad_() for v in names}
    some = {v: s[v].clone().requires_grad_(v not in frozen) for v in names}
    for p in (every, some):
        experts.fed(p["x"], p["gate"], p["up"], p["down"], s["chosen"], weights=p["weights"], base=p["base"]).backward(s["grad"])
    for v in names:
        assert some[v].grad is None if v in frozen else torch.equal(some[v].grad, every[v].grad), v


def test_fed_gradient_that_is_broadcast(experts):  # noqa: F811
    """The gradient of a sum is one value for all elements."""
    s = problem(40, 32, 24, 16, 3, 2, "bf16", 9)
    x = s["x"].clone().requires_grad_()
    experts.fed(x, s["gate"], s["up"], s["down"], s["chosen"], weights=s["weights"]).sum().backward()
    one, pre = torch.ones(40, 16, device="cuda", dtype=torch.bfloat16), experts.feed(s["x"], s["gate"], s["up"], s["down"], s["chosen"], return_pre=True)[1]
    assert torch.equal(x.grad, experts.feed_backward(one, s["x"], s["gate"], s["up"], s["down"], s["chosen"], pre, weights=s["weights"]).x)


def test_feed_python_refusals(experts):  # noqa: F811
    s = problem(6, 16, 24, 32, 3, 2, "bf16", 1)
    m, c = (s["gate"], s["up"], s["down"]), s["chosen"]
    with pytest.raises(ValueError, match="chosen is None"):
        experts.feed(s["x"], *m)
    with pytest.raises(ValueError, match="up has shape"):
        experts.feed(s["x"], m[0], m[1][:2], m[2], c)
    with pytest.raises(ValueError, match="down has shape"):
        experts.feed(s["x"], m[0], m[1], m[2][:, :, :20], c)
    with pytest.raises(ValueError, match="act="):
        experts.feed(s["x"], *m, c, act="tanh")
    with pytest.raises(TypeError, match="chosen"):
        experts.feed(s["x"], *m, c.long())
    with pytest.raises(ValueError, match="contiguous"):
        experts.feed(s["x"], *m, c[:, :1])
    with pytest.raises(ValueError, match="weights"):
        experts.feed(s["x"], *m, c, weights=s["weights"][:, :1])
    with pytest.raises(TypeError, match="gate"):
        experts.feed(s["x"], m[0].half(), m[1], m[2], c)
    with pytest.raises(ValueError, match="side by side"):
        experts.feed(s["x"], m[0].transpose(1, 2).contiguous().transpose(1, 2), m[1], m[2], c)
    with pytest.raises(ValueError, match="base"):
        experts.feed(s["x"], *m, c, base=s["base"][:, :8])
    wide = torch.zeros(6, 40, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="out shares memory with base"):
        experts.feed(s["x"], *m, c, base=wide[:, :32], out=wide[:, 1:33])
    with pytest.raises(RuntimeError, match="overlap"):
        experts.feed(s["x"], *m, c, out=wide[:1, :32].expand(6, 32))
    _, pre = experts.feed(s["x"], *m, c, return_pre=True)
    with pytest.raises(ValueError, match="pre has shape"):
        experts.feed_backward(s["grad"], s["x"], *m, c, pre[:, :1])
    with pytest.raises(ValueError, match="grad has shape"):
        experts.feed_backward(s["grad"][:, :8], s["x"], *m, c, pre)


def check_parts(experts, s, dtype, act="silu"):  # noqa: F811
    """A large problem by some of its rows (out, pre, the gradients of rows and weights are theirs alone) and
    some of its hidden places (the matrices' gradients there are)."""
    x, m, chosen = s["x"], (s["gate"], s["up"], s["down"]), s["chosen"]
    n, f = x.shape[0], m[0].shape[1]
    opt = dict(weights=s["weights"], act=act)
    out, pre = experts.feed(x, *m, chosen, base=s["base"], return_pre=True, **opt)
    assert torch.equal(out, experts.feed(x, *m, chosen, base=s["base"], **opt))
    g = experts.feed_backward(s["grad"], x, *m, chosen, pre, base=s["grad_base"], **opt)
    rows = sorted({*range(0, n, max(1, n // 13)), 15, 16, 63, 64, 127, 128, 255, 256, n - 1} & set(range(n)))
    I, M = chosen.cpu().numpy(), [f64(v) for v in m]
    want = ref.feed(f64(x[rows]), *M, I[rows], f64(s["weights"][rows]), f64(s["base"][rows]), act, dtype, f64(s["grad"][rows]), f64(s["grad_base"][rows]))
    for name, got in (("out", out), ("pre", pre), ("x", g.x), ("weights", g.weights)):
        near(got[rows], *want[name], name)
    places = sorted({*range(0, f, max(1, f // 7)), 31, 32, 127, 128, 255, 256, f - 1} & set(range(f)))
    some = M[0][:, places], M[1][:, places], M[2][:, :, places]
    want = ref.feed(f64(x), *some, I, f64(s["weights"]), None, act, dtype, f64(s["grad"]))
    for name, got in (("gate", g.gate[:, places]), ("up", g.up[:, places]), ("down", g.down[:, :, places])):
        near(got, *want[name], f"grad_{name}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,o,a,k", [(4090, 4088, 4088, 4088, 1, 1), (6000, 2040, 3000, 2040, 3, 1), (2100, 2056, 4104, 2000, 2, 2)])
def test_feed_large(experts, n, d, f, o, a, k, dtype):  # noqa: F811
    """The largest tiles of every product, cut on all sides."""
    print("feed large", n, d, f, o, a, k, dtype, flush=True)
    s = problem(n, d, f, o, a, k, dtype, n)
    if a == 1:
        s["chosen"].clamp_(min=0, max=0)
    check_parts(experts, s, dtype, act="gelu" if a == 1 else "silu")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,o,a,k", [(2500, 64, 4104, 2544, 1, 1), (1800, 72, 4200, 1800, 1, 1), (2500, 2544, 2064, 64, 1, 1), (1200, 2544, 2072, 2536, 1, 2), (2300, 2544, 4104, 2536, 3, 1), (2500, 2540, 2060, 2540, 1, 1)])
def test_feed_sums_in_parts(experts, n, d, f, o, a, k, dtype):  # noqa: F811
    """Sums that are cut over blocks, in two and in four, and joined: where tiles of 256 leave half of the CUs idle."""
    print("feed parts", n, d, f, o, a, k, dtype, flush=True)
    check_parts(experts, problem(n, d, f, o, a, k, dtype, n + d), dtype)


def test_feed_fp32_large(experts):  # noqa: F811
    check_parts(experts, problem(5000, 1000, 2052, 1004, 2, 1, "fp32", 3), "fp32")


def test_feed_out_in_x(experts):  # noqa: F811
    """out one column on in x's rows, and between them: the rows are read before any is written."""
    for n, k in ((2, 2), (300, 1), (300, 2)):
        s = problem(n, 64, 72, 64, 3, k, "bf16", 8)
        m = s["gate"], s["up"], s["down"]
        want = experts.feed(s["x"], *m, s["chosen"], weights=s["weights"], base=s["base"])
        wide = torch.zeros(n, 72, dtype=torch.bfloat16, device="cuda")
        wide[:, :64] = s["x"]
        aligned = experts.feed(wide[:, :64], *m, s["chosen"], weights=s["weights"], base=s["base"])
        assert torch.equal(aligned, want)
        assert torch.equal(experts.feed(wide[:, :64], *m, s["chosen"], weights=s["weights"], base=s["base"], out=wide[:, 1:65]), want)
        both = torch.zeros(n, 128, dtype=torch.bfloat16, device="cuda")
        both[:, :64] = s["x"]
        assert torch.equal(experts.feed(both[:, :64], *m, s["chosen"], weights=s["weights"], base=s["base"], out=both[:, 64:]), want) and torch.equal(both[:, :64], s["x"])
