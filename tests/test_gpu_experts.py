"""The routing and adapter operators on the GPU against their formulas in 64 bits.

Bounds (u = 2^-24, the rounding of fp32; HALF the rounding of a result to its type: u, 2^-8
for bf16 (8 bits), 2^-11 for fp16 (11 bits), whose smallest step is 2^-24):
* a probability is exp of a difference of magnitude at most R, scaled to base 2 (one
  rounding of the difference, one of the product, each worth R u in the result's
  relative error), an exp2 and a reciprocal within a few u, over a sum of e such terms:
  (2 R + log2(e) + 16) u relative, and as much again where two of them meet;
* a sum of m products is off by at most (m + 8) u times the sum of their magnitudes
  in whichever order it is taken;
* with 16-bit types a low-rank vector may enter its second product as two parts of its
  type, which leaves at most 2^-15 of its magnitude out (rows, or for fp16 2^-15 and
  the smallest step).
"""

from __future__ import annotations

import math

import experts_reference as ref
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"fp32": U, "bf16": 2.0**-8, "fp16": 2.0**-11}
STEP = {"fp32": 0.0, "bf16": 0.0, "fp16": 2.0**-24}


@pytest.fixture(scope="module")
def experts():
    from skmetal_amd import _bridge, experts

    if not _bridge.HIP_AVAILABLE:
        pytest.fail(f"GPU path unavailable on a GPU run: {_bridge.last_error()}")
    return experts


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, bound, what):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    want, bound = np.broadcast_to(want, got.shape), np.broadcast_to(bound, got.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        at = tuple(int(v) for v in np.argwhere(bad)[0])
        pytest.fail(f"{what}: {bad.sum()} of {bad.size} off, first at {at}: {got[at]} for {want[at]}, off {off[at]}, bound {bound[at]}")


# ---- route ----


def scores(n, e, kind, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, e, generator=g) * 2
    if kind == "ties":
        z = torch.randint(-2, 3, (n, e), generator=g).float() * 0.5
        z[z == 0] = torch.where(torch.rand(int((z == 0).sum()), generator=g) < 0.5, -0.0, 0.0)
    elif kind == "equal":
        z = torch.full((n, e), -7.25)
    elif kind == "excluded":
        z[torch.rand(n, e, generator=g) < 0.3] = -math.inf
        z[torch.rand(n, e, generator=g) < 0.05] = math.nan
        if n > 2:
            z[n // 2] = -math.inf
    elif kind == "lowest":  # the masking value of many programs: the type's lowest number
        low = torch.finfo(dtype).min
        z[torch.rand(n, e, generator=g) < 0.5] = low
        if n > 2:
            z[n // 2] = low
    elif kind == "far":
        z = z * 20
    return z.to(dtype)


ROUTES = [(1, 1, 1), (1, 64, 2), (3, 2, 2), (5, 37, 3), (257, 64, 16), (130, 256, 8), (65, 257, 4), (33, 1000, 6), (9, 2048, 16), (4097, 8, 1), (70, 300, 5),
          (19, 65, 9), (2050, 16, 4), (12, 513, 12), (6, 1025, 1)]


def check_route(experts, z, k, mask, normalize, dtype, dw=None, dl=None):
    r = experts.route(z, k, mask=mask, normalize=normalize)
    zz, n, e = f64(z), *z.shape
    m = None if mask is None else mask.cpu().numpy().astype(bool)
    w, ex, counts, sums, rows, loss, p = ref.route(zz, k, m, normalize)
    fin = np.where(np.isfinite(zz), zz, np.nan)
    span = np.nan_to_num(np.nanmax(fin) - np.nanmin(fin)) if np.isfinite(fin).any() else 0.0
    span = min(span, 110.0)  # beyond exp's range the probability is 0 within 2^-126
    rel = 2 * (2 * span + math.log2(e) + 16) * U
    np.testing.assert_array_equal(r.experts.cpu().numpy(), ex)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), counts)
    assert r.rows.tolist() == [rows] and r.loss.shape == ()
    near(r.weights, w, rel * w + 2.0**-120, "weights")
    near(r.prob_sums, sums, (rel + (n + 8) * U) * sums + 2.0**-120, "prob_sums")
    near(r.loss, np.float64(loss), (rel + (n + 8) * U) * loss, "loss")
    if dw is None and dl is None:
        return r
    got = experts.route_backward(z, r, grad_weights=dw, grad_loss=dl, mask=mask, normalize=normalize)
    want, mag = ref.route_backward(p, w, ex, counts, rows, np.zeros((n, k)) if dw is None else f64(dw), 0.0 if dl is None else float(dl), normalize)
    name = {v: k for k, v in TYPES.items()}[dtype]
    assert got.dtype == dtype and got.shape == z.shape
    near(got, want, 2 * (rel + (e + k + 8) * U) * mag + HALF[name] * np.abs(want) + STEP[name] + 2.0**-120, "grad_logits")
    return r


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,e,k", ROUTES)
def test_route(experts, n, e, k, dtype):
    print("route", n, e, k, dtype, flush=True)
    z = scores(n, e, "normal", TYPES[dtype], n + e).cuda()
    g = torch.Generator().manual_seed(3)
    dw, dl = torch.randn(n, k, generator=g).cuda(), torch.tensor(0.7 * n, device="cuda")
    check_route(experts, z, k, None, (n + k) % 2 == 0, TYPES[dtype], dw, dl)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["ties", "equal", "excluded", "lowest", "far"])
@pytest.mark.parametrize("n,e,k", [(1, 5, 5), (37, 24, 4), (300, 256, 8), (21, 700, 16)])
def test_route_hard_scores(experts, n, e, k, kind, dtype):
    print("route", kind, n, e, k, dtype, flush=True)
    z = scores(n, e, kind, TYPES[dtype], n).cuda()
    g = torch.Generator().manual_seed(4)
    mask = (torch.rand(n, generator=g) < 0.8).cuda()
    dw, dl = torch.randn(n, k, generator=g).cuda(), torch.tensor(1.3, device="cuda")
    for normalize in (False, True):
        check_route(experts, z, k, None, normalize, TYPES[dtype], dw, dl)
        check_route(experts, z, k, mask, normalize, TYPES[dtype], dw, None)
        check_route(experts, z, k, mask, normalize, TYPES[dtype], None, dl)


def test_route_masked_rows_hold_anything(experts):
    z = scores(50, 40, "normal", torch.float32, 1)
    mask = torch.arange(50) % 3 != 0
    clean = z.clone()
    z[~mask] = math.nan
    z[0] = math.inf
    a, b = (experts.route(t.cuda(), 4, mask=mask.cuda()) for t in (z, clean))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    dw = torch.ones(50, 4, device="cuda")
    dw[0] = math.nan  # a gradient in a place that holds no expert
    g = experts.route_backward(z.cuda(), a, grad_weights=dw, grad_loss=torch.ones((), device="cuda"), mask=mask.cuda())
    assert torch.isfinite(g).all() and (g[~mask.cuda()] == 0).all()


def test_route_every_row_masked_and_no_rows(experts):
    z = scores(7, 12, "normal", torch.bfloat16, 1).cuda()
    r = experts.route(z, 3, mask=torch.zeros(7, dtype=torch.bool, device="cuda"))
    assert (r.experts == -1).all() and (r.weights == 0).all() and r.loss.item() == 0 and r.rows.item() == 0 and (r.counts == 0).all() and (r.prob_sums == 0).all()
    g = experts.route_backward(z, r, grad_loss=torch.ones((), device="cuda"), mask=torch.zeros(7, dtype=torch.bool, device="cuda"))
    assert (g == 0).all()
    r = experts.route(z[:0], 3)
    assert r.experts.shape == (0, 3) and r.loss.item() == 0 and (r.counts == 0).all() and (r.prob_sums == 0).all() and r.rows.item() == 0
    assert experts.route_backward(z[:0], r, grad_loss=torch.ones((), device="cuda")).shape == (0, 12)


def test_route_strided_rows_and_masks(experts):
    wide = scores(60, 64, "normal", torch.bfloat16, 9).cuda()
    for view in (wide[:, :33], wide[:, 3:40], wide[::2, 1:], wide.as_strided((60, 20), (0, 1))):
        check_route(experts, view, 3, None, True, torch.bfloat16, torch.ones(view.shape[0], 3, device="cuda"), None)
    mask = torch.arange(120, device="cuda") % 5 != 0
    check_route(experts, wide, 2, mask[::2], False, torch.bfloat16, None, torch.tensor(2.0, device="cuda"))


def test_route_same_bits_every_time(experts):
    z = scores(5000, 96, "normal", torch.bfloat16, 5).cuda()
    a = experts.route(z, 4)
    for _ in range(3):
        for x, y in zip(a, experts.route(z, 4)):
            assert torch.equal(x, y)


def test_route_gradient_is_the_loss_difference(experts):
    """Central differences of the kernel's own loss and weights along a direction that
    changes no choice: truncation h^2 and rounding U / h, under 2e-3 of the slope here."""
    n, e, k = 64, 16, 2
    g = torch.Generator().manual_seed(8)
    z = torch.stack([torch.randperm(e, generator=g) for _ in range(n)]).float() * 0.25
    v = torch.rand(n, e, generator=g) - 0.5
    dw = torch.randn(n, k, generator=g).cuda()
    h = 0.03125
    for normalize in (False, True):
        r = experts.route(z.cuda(), k, normalize=normalize)
        grad = experts.route_backward(z.cuda(), r, grad_weights=dw, grad_loss=torch.tensor(float(n), device="cuda"), normalize=normalize)
        side = []
        for s in (h, -h):
            q = experts.route((z + s * v).cuda(), k, normalize=normalize)
            assert torch.equal(q.experts, r.experts)
            side.append(float((q.weights * dw).double().sum()) + n * float(q.loss))
        slope = float((grad.cpu().double() * v.double()).sum())
        scale = float((grad.cpu().double().abs() * v.double().abs()).sum())
        assert abs((side[0] - side[1]) / (2 * h) - slope) < 2e-3 * scale


# ---- adapt ----


def problem(n, d, o, r, a, dtype, seed, law="rows"):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    ids = torch.randint(-1, a + 1, (n,), generator=g)  # -1 and a: none
    if law == "runs":
        ids = ids.sort().values
    elif law == "one":
        ids = torch.full((n,), max(0, a - 1))
    elif law == "none":
        ids = torch.full((n,), -1)
    elif law == "wild":
        ids[torch.rand(n, generator=g) < 0.3] = -(2**31)
        ids[torch.rand(n, generator=g) < 0.3] = 2**31 - 1
    return dict(x=torch.randn(n, d, generator=g).to(t).cuda(), down=(torch.randn(a, r, d, generator=g) / math.sqrt(d)).to(t).cuda(),
                up=(torch.randn(a, r, o, generator=g) / math.sqrt(r)).to(t).cuda(), ids=ids.int().cuda(), base=torch.randn(n, o, generator=g).to(t).cuda(),
                gates=torch.randn(n, generator=g).cuda(), scales=(torch.rand(a, generator=g) + 0.5).cuda(), grad=torch.randn(n, o, generator=g).to(t).cuda(),
                grad_base=torch.randn(n, d, generator=g).to(t).cuda())


def part(dtype):
    return 0.0 if dtype == "fp32" else 2.0**-15


def check_adapt(experts, s, dtype, gates=True, scales=True, base=True, backward=True, **kw):
    x, down, up, ids = s["x"], s["down"], s["up"], s["ids"]
    (n, d), (a, r, o) = x.shape, up.shape
    opt = dict(gates=s["gates"] if gates else None, scales=s["scales"] if scales else None)
    npo = {k: None if v is None else f64(v) for k, v in opt.items()}
    X, A, B, I = f64(x), f64(down), f64(up), ids.cpu().numpy()
    out, low = experts.adapt(x, down, up, ids, base=s["base"] if base else None, return_low=True, **opt, **kw)
    bare = experts.adapt(x, down, up, ids, base=s["base"] if base else None, **opt)
    assert torch.equal(out, bare)
    want, wlow, mag = ref.adapt(X, A, B, I, f64(s["base"]) if base else None, **npo)
    lowmag = np.zeros_like(wlow)
    for q in range(a):
        lowmag[I == q] = np.abs(X[I == q]) @ np.abs(A[q]).T
    near(low, wlow, (d + 8) * U * lowmag, "low")
    half, step = HALF[dtype], STEP[dtype]
    near(out, want, ((d + r + 16) * U + part(dtype)) * mag + 2 * U * np.abs(want) + half * np.abs(want) + step, "out")
    if not backward:
        return out
    g = experts.adapt_backward(s["grad"], x, down, up, ids, low, base=s["grad_base"] if base else None, **opt)
    again = experts.adapt_backward(s["grad"], x, down, up, ids, low, base=s["grad_base"] if base else None, **opt)
    (dx, dA, dB, dg), (mx, mA, mB, mg) = ref.adapt_backward(f64(s["grad"]), X, A, B, I, f64(s["grad_base"]) if base else None, **npo)
    most = int(np.bincount(I[(I >= 0) & (I < a)], minlength=1).max()) if n else 0
    p = part(dtype)
    near(g.x, dx, ((o + r + 16) * U + p) * mx + 2 * U * np.abs(dx) + half * np.abs(dx) + step, "grad_x")
    near(g.down, dA, ((o + most + 16) * U + p) * mA + half * np.abs(dA) + step, "grad_down")
    near(g.up, dB, ((d + most + 16) * U + p) * mB + half * np.abs(dB) + step, "grad_up")
    if gates:
        near(g.gates, dg, (d + o + r + 16) * U * mg, "grad_gates")
    else:
        assert g.gates is None
    for p1, p2 in zip(g, again):
        assert p1 is p2 is None or torch.equal(p1, p2)
    return out


ADAPTS = [(1, 1024, 1024, 8, 16), (7, 33, 65, 5, 3), (64, 256, 256, 16, 4), (130, 520, 96, 33, 2), (65, 64, 64, 128, 2), (300, 100, 100, 1, 40), (3, 1, 1, 1, 1),
          (1000, 48, 40, 12, 1), (513, 264, 136, 16, 70), (33, 2056, 8, 64, 5), (2100, 64, 72, 20, 300), (17, 8, 2048, 17, 2)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,o,r,a", ADAPTS)
def test_adapt(experts, n, d, o, r, a, dtype):
    print("adapt", n, d, o, r, a, dtype, flush=True)
    check_adapt(experts, problem(n, d, o, r, a, dtype, n + d), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,o,r,a", [(600, 200, 136, 128, 3), (1200, 1032, 520, 40, 6), (17000, 24, 16, 4, 9), (3000, 40, 48, 70, 2048), (33000, 16, 8, 16, 30),
                                       (512, 64, 64, 16, 5), (900, 4096, 40, 64, 2), (5000, 72, 520, 33, 4)])
def test_adapt_sorted_rows(experts, n, d, o, r, a, dtype):
    """Calls that sort their rows: several segments, chunks of an adapter, every size of tile."""
    print("adapt", n, d, o, r, a, dtype, flush=True)
    check_adapt(experts, problem(n, d, o, r, a, dtype, n + d), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,o,r,a", [(40, 1500, 2100, 9, 4), (3, 2048, 24, 32, 2), (3, 2049, 24, 32, 2), (200, 700, 1100, 17, 6), (20, 24, 300, 60, 3), (2, 12, 4096, 16, 1),
                                       (12, 4100, 70, 16, 3), (300, 72, 513, 33, 7), (65, 1024, 1024, 16, 9), (70, 1024, 1000, 64, 4), (300, 1024, 8, 49, 3)])
def test_adapt_few_rows(experts, n, d, o, r, a, dtype):
    """Calls on either side of where both products become one launch."""
    print("adapt", n, d, o, r, a, dtype, flush=True)
    check_adapt(experts, problem(n, d, o, r, a, dtype, n + d), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("law", ["runs", "one", "none", "wild"])
@pytest.mark.parametrize("n,d,o,r,a", [(40, 72, 48, 6, 4), (700, 160, 64, 16, 5), (1500, 65, 33, 9, 90)])
def test_adapt_ids(experts, n, d, o, r, a, law, dtype):
    print("adapt", law, n, d, o, r, a, dtype, flush=True)
    check_adapt(experts, problem(n, d, o, r, a, dtype, n + d, law), dtype)


@pytest.mark.parametrize("gates", [False, True])
@pytest.mark.parametrize("scales", [False, True])
@pytest.mark.parametrize("base", [False, True])
def test_adapt_options(experts, gates, scales, base):
    for dtype, n in (("bf16", 5), ("fp32", 300), ("bf16", 400)):
        check_adapt(experts, problem(n, 96, 80, 8, 6, dtype, 21), dtype, gates, scales, base)


def test_adapt_strides_and_places(experts):
    """Rows apart, rows that start off any 16-byte line, adapters cut out of larger ones,
    ids and gates as columns of a matrix, and out in base's place."""
    for dtype in TYPES:
        for n in (9, 333):
            s = problem(n, 101, 90, 12, 5, dtype, 6)
            wide = problem(n, 160, 128, 16, 7, dtype, 7)
            s["x"], s["base"] = wide["x"][:, 3:104], wide["base"][:, 5:95]
            s["grad"], s["grad_base"] = wide["grad"][:, 1:91], wide["grad_base"][:, 7:108]
            s["down"], s["up"] = wide["down"][1:6, 2:14, 9:110], wide["up"][1:6, 2:14, 11:101]
            s["ids"] = torch.stack([s["ids"], s["ids"] + 1], 1)[:, 0]
            s["gates"] = torch.stack([s["gates"], s["gates"]], 1)[:, 1]
            want = check_adapt(experts, s, dtype)
            place = torch.full((n, 128), 3.0, dtype=TYPES[dtype], device="cuda")
            place[:, 5:95] = s["base"]
            got = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=place[:, 5:95], gates=s["gates"], scales=s["scales"], out=place[:, 5:95])
            assert got.data_ptr() == place[:, 5:95].data_ptr() and torch.equal(got, want)
            assert (place[:, :5] == 3).all() and (place[:, 95:] == 3).all()


def test_adapt_broadcast_rows(experts):
    s = problem(50, 64, 48, 8, 3, "bf16", 6)
    s["x"] = s["x"][:1].expand(50, 64)
    s["base"] = s["base"][:1].expand(50, 48)
    s["gates"] = s["gates"][:1].expand(50)
    check_adapt(experts, s, "bf16")


def test_adapt_nothing_to_do(experts):
    s = problem(0, 16, 24, 4, 3, "bf16", 1)
    check_adapt(experts, s, "bf16")
    s = problem(20, 16, 24, 4, 0, "bf16", 1)
    out, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"], return_low=True)
    assert torch.equal(out, s["base"]) and (low == 0).all()
    g = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, base=s["grad_base"], gates=s["gates"])
    assert torch.equal(g.x, s["grad_base"]) and g.down.shape == (0, 4, 16) and (g.gates == 0).all()


def test_adapt_rows_without_an_adapter_touch_nothing(experts):
    """NaN and infinity in x, gates or low of rows without an adapter, and in adapters
    that no row has, stay where they are."""
    for n in (11, 600):
        s = problem(n, 64, 48, 8, 4, "bf16", 13)
        s["ids"][s["ids"] == 2] = 0
        none = (s["ids"] < 0) | (s["ids"] >= 4)
        for name in ("x", "gates", "grad"):
            s[name][none] = math.nan
        s["down"][2], s["up"][2], s["scales"][2] = math.inf, math.nan, math.nan
        opt = dict(gates=s["gates"], scales=s["scales"])
        out, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"], return_low=True, **opt)
        assert torch.isfinite(out).all() and torch.equal(out[none], s["base"][none]) and (low[none] == 0).all()
        g = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, base=s["grad_base"], **opt)
        assert all(torch.isfinite(t).all() for t in g) and torch.equal(g.x[none], s["grad_base"][none])
        assert (g.down[2] == 0).all() and (g.up[2] == 0).all() and (g.gates[none] == 0).all()


def test_adapt_large_values_pass_through(experts):
    """An infinity in a row's own x reaches that row alone."""
    for n in (8, 500):
        s = problem(n, 64, 48, 8, 4, "bf16", 14)
        s["ids"][:] = torch.arange(n, device="cuda").int() % 4
        plain = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"])
        s["x"][5, 3] = math.inf
        out = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"])
        rest = torch.arange(n, device="cuda") != 5
        assert not torch.isfinite(out[5]).all() and torch.equal(out[rest], plain[rest])


def test_adapt_gradient_is_the_difference(experts):
    """out is linear in each of x, down, up and gates: one-sided differences with a step of
    1 are exact but for rounding ((d + o + r) U of the magnitudes)."""
    s = problem(40, 32, 24, 4, 3, "fp32", 15)
    opt = dict(scales=s["scales"])

    def value(**kw):
        v = {**{k: s[k] for k in ("x", "down", "up", "gates")}, **kw}
        out = experts.adapt(v["x"], v["down"], v["up"], s["ids"], gates=v["gates"], **opt)
        return float((out.double() * s["grad"].double()).sum()), float((out.double().abs() * s["grad"].double().abs()).sum())

    _, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], gates=s["gates"], return_low=True, **opt)
    g = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, gates=s["gates"], **opt)
    at, scale0 = value()
    gen = torch.Generator().manual_seed(2)
    for name in ("x", "down", "up", "gates"):
        v = torch.randn(s[name].shape, generator=gen).cuda()
        moved, scale1 = value(**{name: s[name] + v})
        slope = float((getattr(g, name).double() * v.double()).sum())
        assert abs(moved - at - slope) < 64 * (32 + 24 + 4) * U * (scale0 + scale1)


# ---- together ----


def test_autograd(experts):
    torch.manual_seed(0)
    n, d, o, r, e, k = 90, 32, 24, 4, 6, 2
    x = torch.randn(n, d, device="cuda", requires_grad=True)
    centres = torch.randn(e, d, device="cuda", requires_grad=True)
    down, up = (torch.randn(e, r, w, device="cuda", requires_grad=True) for w in (d, o))
    W = torch.randn(d, o, device="cuda", requires_grad=True)
    logits = x @ centres.T.contiguous() * 0.1
    q = experts.routed(logits, k, normalize=True)
    y = x @ W
    for t in range(k):
        y = experts.adapted(x, down, up, q.experts[:, t], base=y, gates=q.weights[:, t])
    loss = y.square().mean() + 0.1 * q.loss
    got = torch.autograd.grad(loss, [x, centres, down, up, W])
    x2, c2, A2, B2, W2 = (v.detach().double().requires_grad_() for v in (x, centres, down, up, W))
    p = torch.softmax(x2 @ c2.T * 0.1, 1)
    take = q.experts.long()
    w = p.gather(1, take)
    w = w / w.sum(1, keepdim=True)
    y2 = x2 @ W2
    for t in range(k):
        low = (A2[take[:, t]] * x2[:, None, :]).sum(2)
        y2 = y2 + w[:, t, None] * (B2[take[:, t]] * low[:, :, None]).sum(1)
    counts = torch.bincount(take.flatten(), minlength=e).double()
    loss2 = y2.square().mean() + 0.1 * e / (k * n * n) * (counts * p.sum(0)).sum()
    want = torch.autograd.grad(loss2, [x2, c2, A2, B2, W2])
    assert abs(loss.item() - loss2.item()) < 1e-5 * abs(loss2.item())
    for a, b in zip(got, want):  # fp32 chains of under 200 terms, 2^-24 each: 1e-5 of the norm
        assert float((a.double() - b).norm()) < 1e-4 * float(b.norm())


def test_another_stream_and_a_graph(experts):
    s = problem(700, 128, 96, 16, 5, "bf16", 3)
    z = scores(700, 40, "normal", torch.bfloat16, 2).cuda()

    def work():
        r = experts.route(z, 2, normalize=True)
        out, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"], gates=r.weights[:, 0], return_low=True)
        g = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, gates=r.weights[:, 0])
        return [*r, out, *g, experts.route_backward(z, r, grad_weights=r.weights, grad_loss=r.loss, normalize=True)]

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
    for i in range(4):  # each replay on new inputs, beside eager work
        s["x"].copy_(torch.randn_like(s["x"].float()))
        z.copy_(torch.randn_like(z.float()))
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), i


def test_python_refusals(experts):
    z = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    A, B = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 6, device="cuda")
    with pytest.raises(ValueError, match="top_k"):
        experts.route(z, 9)
    with pytest.raises(ValueError, match="top_k"):
        experts.route(torch.zeros(4, 40, device="cuda"), 17)
    with pytest.raises(ValueError, match="experts"):
        experts.route(torch.zeros(4, 4096, device="cuda"), 2)
    with pytest.raises(ValueError, match="side by side"):
        experts.route(z.T, 2)
    with pytest.raises(ValueError, match="dimensions"):
        experts.route(z[0], 2)
    with pytest.raises(TypeError, match="mask"):
        experts.route(z, 2, mask=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="mask"):
        experts.route(z, 2, mask=torch.ones(5, dtype=torch.bool, device="cuda"))
    r = experts.route(z, 2)
    with pytest.raises(ValueError, match="grad_weights"):
        experts.route_backward(z, r, grad_weights=torch.zeros(4, 3, device="cuda"))
    with pytest.raises(TypeError, match="grad_loss"):
        experts.route_backward(z, r, grad_loss=torch.zeros((), dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="columns"):
        experts.adapt(z, B, A, ids)
    with pytest.raises(ValueError, match="agree"):
        experts.adapt(z, A, B[:, :2], ids)
    with pytest.raises(TypeError, match="ids"):
        experts.adapt(z, A, B, ids.long())
    with pytest.raises(ValueError, match="ids"):
        experts.adapt(z, A, B, ids[:3])
    with pytest.raises(TypeError, match="down"):
        experts.adapt(z, A.half(), B, ids)
    with pytest.raises(ValueError, match="base"):
        experts.adapt(z, A, B, ids, base=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(ValueError, match="on cpu"):
        experts.adapt(z, A, B, ids.cpu())
    with pytest.raises(ValueError, match="rank"):
        experts.adapt(z, torch.zeros(1, 129, 8, device="cuda"), torch.zeros(1, 129, 6, device="cuda"), ids)
    with pytest.raises(RuntimeError, match="overlap"):
        experts.adapt(z, A, B, ids, out=torch.zeros(6, device="cuda").expand(4, 6))
    with pytest.raises(ValueError, match="low"):
        experts.adapt_backward(torch.zeros(4, 6, device="cuda"), z, A, B, ids, torch.zeros(4, 2, device="cuda"))


def test_cluster_experts_example(experts):
    """The whole path: a KMeans fit's centres as router, training steps, served rows.  The
    fit brings the loss down, and a served row is the training pass's own (bf16: the same
    products in another split of the sums, a few roundings of 2^-8)."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "cluster_experts.py"
    spec = importlib.util.spec_from_file_location("cluster_experts", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, net, x = example.main(["--rows", "3000", "--width", "64", "--experts", "8", "--steps", "40"])
    assert losses[-1] < 0.7 * losses[0]
    with torch.no_grad():
        y, _ = net(x)
    for n in (1, 5, 200):
        off = (net.serve(x[:n]).float() - y[:n].float()).abs()
        assert float(off.max()) <= 4 * 2.0**-8 * float(y.float().abs().max())


def test_labels_are_adapter_ids(experts):
    """A cluster's rows through its adapter: KMeans labels as they come."""
    from sklearn.cluster import KMeans

    import skmetal_amd

    s = problem(1500, 24, 32, 4, 5, "fp32", 4)
    model = skmetal_amd.accelerate(KMeans(n_clusters=5, n_init=1, random_state=0)).fit(s["x"].cpu().numpy())
    assert model.labels_.dtype == np.int32
    s["ids"] = torch.from_numpy(model.labels_).cuda()
    check_adapt(experts, s, "fp32")


def test_sizes_around_the_kernels_choices(experts):
    """Rows around the steps from one block to several (route) and from no sort to a sort."""
    for n in (127, 128, 129, 1023, 1025):
        check_route(experts, scores(n, 200, "normal", torch.bfloat16, n).cuda(), 4, None, True, torch.bfloat16, torch.ones(n, 4, device="cuda"), None)
    for e in (8, 9, 32, 33, 64, 65, 256, 257, 512, 513, 1024):
        check_route(experts, scores(40, e, "ties", torch.float16, e).cuda(), min(e, 8), None, False, torch.float16, None, torch.tensor(1.0, device="cuda"))
    for n in (511, 512, 513):
        check_adapt(experts, problem(n, 64, 64, 16, 5, "bf16", n), "bf16")
    for n in (64, 65):  # 2^25 and 2^24 products
        check_adapt(experts, problem(n, 4096, 4096, 64, 3, "bf16", n), "bf16")
