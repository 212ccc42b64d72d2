"""Log probabilities and dropout on the GPU against their formulas in 64 bits.

Bounds (u = 2^-24): with m the row's largest score and R the magnitude of the differences z - m that count (at
most 200), a term exp(z - m) is off by (R + 4) u of itself, and so is every step to a new maximum; a lane adds up at most v
/ 64 + 32 terms and steps one after another.  So S is off by rel = (2 R + 2 (v / 64 + 32)) u of itself, ln S by that and its
own rounding, T by as much of its terms' magnitude."""

from __future__ import annotations

import math

import feed_reference as ref
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import HALF, STEP, TYPES, U, experts, f64, near, scores  # noqa: E402, F401 -- a fixture

pytestmark = pytest.mark.gpu


def check(experts, z, targets, k, dtype, backward=True):  # noqa: F811
    n, v = z.shape
    zz, t = f64(z), targets.cpu().numpy().astype(np.int64)
    lp, ent, lse, top, toplp, p, logp = ref.rate(zz, t, k)
    r = experts.rate(z, targets, top_k=k)
    fin = np.where(np.isfinite(zz), zz, np.nan)
    with np.errstate(all="ignore"):
        m = np.nan_to_num(np.nanmax(np.where(np.isfinite(fin), fin, -np.inf), axis=1), neginf=0.0)
    d = np.where(np.isfinite(zz), zz - m[:, None], 0.0)
    span = min(200.0, float(np.abs(d).max())) if n else 0.0
    rel = (2 * span + 2 * (v / 64 + 32)) * U
    mean = (p * np.abs(d)).sum(1)  # E|z - m|
    fine = np.isfinite(lse)
    logs = np.where(fine, np.nan_to_num(lse) - m, 0.0)
    at = lambda b: np.where(fine, b, 2.0**-120)  # noqa: E731

    def same(got, want, bound, what):
        got = f64(got) if isinstance(got, torch.Tensor) else got
        assert np.array_equal(np.isnan(got), np.isnan(want)), what
        assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]) and np.isfinite(got[np.isfinite(want)]).all(), what
        ok = np.isfinite(want)
        near(got[ok], want[ok], np.broadcast_to(bound, want.shape)[ok], what)

    has = (t >= 0) & (t < v)
    dt = np.where(has, np.abs(np.where(np.isfinite(lp), lp, 0.0) + logs), 0.0)
    same(r.log_probs, lp, at(rel + 4 * U * (dt + np.abs(logs)) + 2.0**-100), "log_probs")
    same(r.entropy, ent, at(rel * (2 + 3 * mean) + 8 * U * (np.abs(logs) + mean) + 2.0**-100), "entropy")
    same(r.lse, lse, at(rel + 4 * U * (np.abs(m) + np.abs(logs)) + 2.0**-100), "lse")
    with np.errstate(invalid="ignore"):
        both = np.where(fine, f64(r.lse) + f64(r.lse_rest), lse)
    same(both, lse, at(rel + 4 * U * np.abs(logs) + 2.0**-46 * np.abs(m) + 2.0**-100), "lse + lse_rest")
    if k:
        np.testing.assert_array_equal(r.top.cpu().numpy(), top)
        # a named score may lie as far under m as it likes: its difference and the result are rounded at their own sizes
        size = np.abs(np.where(np.isfinite(toplp), toplp, 0.0))
        same(r.top_log_probs, toplp, at(rel + 4 * U * np.abs(logs) + 2.0**-100)[:, None] + 4 * U * size, "top_log_probs")
    else:
        assert r.top is r.top_log_probs is None
    again = experts.rate(z, targets, top_k=k)
    for a, b in zip(r, again):
        assert a is b is None or torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)
    if not backward:
        return r
    g = torch.Generator().manual_seed(5)
    grads = [torch.randn(n, generator=g) for _ in range(3)]
    for use in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        got = experts.rate_backward(z, targets, r, **{name: v.cuda() for name, v, u in zip(("grad_log_probs", "grad_entropy", "grad_lse"), grads, use) if u})
        gl, ge, gs = (f64(v) * u for v, u in zip(grads, use))
        ent0 = np.where(np.isfinite(ent), ent, 0.0)
        dz, mag = ref.rate_backward(np.nan_to_num(p), np.where(np.isfinite(logp), logp, -np.inf), ent0, t, gl, ge, gs)
        big = np.abs(np.where(np.isfinite(logp), logp, 0.0))
        off = mag * (2 * (rel + 8 * U * (1 + big)) + 8 * U) + np.nan_to_num(p) * np.abs(ge)[:, None] * (rel * (3 + 4 * mean) + 16 * U * (np.abs(logs) + mean))[:, None]
        # exp's results under 2^-126 are 0: a p that small is lost, with the factor that it has in dz
        off = off + 2.0**-126 * (np.abs(gs) + np.abs(gl) + np.abs(ge * ent0))[:, None] + 2.0**-126 * np.abs(ge)[:, None] * big
        rows = lse < np.inf
        assert got.shape == z.shape and got.dtype == z.dtype
        near(f64(got)[rows], dz[rows], (off + HALF[dtype] * np.abs(dz) + STEP[dtype] + 2.0**-120)[rows], "grad_logits")
        assert not rows.size or np.isnan(f64(got)[~rows][zz[~rows] > -np.inf]).all() and (f64(got)[~rows][~(zz[~rows] > -np.inf)] == 0).all()
    return r


def targets_of(n, v, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.where(torch.rand(n, generator=g) < 0.2, torch.tensor([-100, -1, v, 2**31 - 1])[torch.randint(0, 4, (n,), generator=g)],
                       torch.randint(0, v, (n,), generator=g)).int().cuda()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 5, 5), (3, 64, 2), (200, 37, 3), (9, 2048, 16), (7, 2049, 16), (5, 2050, 0), (1, 32_000, 5), (33, 4097, 1), (2, 50_257, 16),
                                   (1100, 5000, 4), (65, 1000, 7)])
def test_rate(experts, n, v, k, dtype):  # noqa: F811
    print("rate", n, v, k, dtype, flush=True)
    check(experts, scores(n, v, "normal", TYPES[dtype], n + v).cuda(), targets_of(n, v, n), k, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["ties", "equal", "excluded", "lowest", "far"])
@pytest.mark.parametrize("n,v,k", [(1, 9, 9), (40, 300, 16), (3, 9000, 16), (20, 2500, 3)])
def test_rate_hard_scores(experts, n, v, k, kind, dtype):  # noqa: F811
    print("rate", kind, n, v, k, dtype, flush=True)
    check(experts, scores(n, v, kind, TYPES[dtype], n + v).cuda(), targets_of(n, v, n), k, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v", [50, 2000, 9000, 70_000])
def test_rate_orders(experts, v, dtype):  # noqa: F811
    """Rows that rise, fall, hold their largest scores on one lane, or hold few scores at all."""
    print("rate orders", v, dtype, flush=True)
    t = TYPES[dtype]
    z = torch.zeros(6, v)
    z[0] = torch.linspace(-9, 9, v)
    z[1] = torch.linspace(9, -9, v)
    z[2] = torch.where(torch.arange(v) % 2048 < 8, 3.0, 0.0) + torch.arange(v) / v  # every 256 lanes' first vectors
    z[3, :] = -math.inf
    z[3, v // 2] = 1.0
    z[4, :] = -math.inf
    z[5, :] = math.nan
    z[5, -3:] = torch.tensor([-1e4, 2.0, 2.0])
    check(experts, z.to(t).cuda(), torch.tensor([0, v - 1, 3, v // 2, 1, v - 1]).int().cuda(), min(16, v), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("v,k", [(70, 16), (2000, 1), (2000, 16), (4100, 3), (70_000, 16)])
def test_rate_few_distinct_scores(experts, v, k, sign, dtype):  # noqa: F811
    """Which of the same scores are named: those of the lowest places, below 0 too."""
    print("rate few distinct", v, k, sign, dtype, flush=True)
    g = torch.Generator().manual_seed(v + k)
    z = sign * torch.tensor([1.0, 1.5, 2.0, 0.0])[torch.randint(0, 3, (5, v), generator=g)]
    z[1] = sign * 2.0
    z[2] = sign * (2.0 + sign)
    z[2, -5:] = sign * 2.0 + 1.0  # five at the end before all others
    z[3, : v // 2] = -math.inf
    z[4, 64:] = -math.inf
    check(experts, z.to(TYPES[dtype]).cuda(), torch.tensor([0, v - 1, 3, v // 2, 1]).int().cuda(), k, dtype)


def test_rate_longest_row(experts):  # noqa: F811
    """The largest row: places up to the last, the same scores at both ends."""
    v = 1 << 22
    z = torch.zeros(1, v)
    z[0, : 1 << 20] = -1.0
    z[0, -3:] = torch.tensor([2.0, 3.0, 3.0])
    z[0, 5] = 3.0
    print("rate longest", flush=True)
    check(experts, z.bfloat16().cuda(), torch.tensor([v - 1]).int().cuda(), 16, "bf16", backward=False)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rate_infinite_scores(experts, dtype):  # noqa: F811
    z = scores(8, 300, "normal", TYPES[dtype], 2)
    z[1, 7] = math.inf
    z[3, 2] = z[3, 200] = math.inf
    z[3, 5] = -math.inf
    z[6] = math.inf
    check(experts, z.cuda(), torch.tensor([0, 7, 7, 5, 1, 2, 3, -1]).int().cuda(), 4, dtype)


def test_rate_large_scores_keep_their_probabilities(experts):  # noqa: F811
    """Scores of 1e5, where an lse in fp32 alone would leave p a hundredth off."""
    z = scores(20, 500, "normal", torch.float32, 8).cuda() + 1e5
    t = targets_of(20, 500, 8)
    check(experts, z, t, 3, "fp32")


def test_rate_strided_rows(experts):  # noqa: F811
    wide = scores(60, 3000, "normal", torch.bfloat16, 9).cuda()
    for view in (wide[:, :2999], wide[:, 3:2500], wide[::2, 1:], wide.as_strided((60, 2500), (0, 1)), wide[:, 5:6]):
        t = targets_of(120, view.shape[1], 1)[: 2 * view.shape[0] : 2]
        check(experts, view, t, 1, "bf16")


def test_rate_nothing_to_do(experts):  # noqa: F811
    z, t = torch.zeros(0, 40, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    r = experts.rate(z, t, top_k=3)
    assert r.log_probs.shape == (0,) and r.top.shape == (0, 3)
    assert experts.rate_backward(z, t, r, grad_lse=torch.zeros(0, device="cuda")).shape == (0, 40)


def test_rate_gradient_is_the_difference(experts):  # noqa: F811
    """Central differences of the kernel's own results along a direction: truncation h^2 and
    rounding u / h of the magnitudes, under 2e-3 of the slope's."""
    n, v, h = 40, 300, 0.03125
    g = torch.Generator().manual_seed(8)
    z, d, w = torch.randn(n, v, generator=g), torch.rand(n, v, generator=g) - 0.5, torch.randn(3, n, generator=g).double().cuda()
    t = targets_of(n, v, 3)
    r = experts.rate(z.cuda(), t)
    grad = experts.rate_backward(z.cuda(), t, r, grad_log_probs=w[0].float(), grad_entropy=w[1].float(), grad_lse=w[2].float())
    side = []
    for s in (h, -h):
        q = experts.rate((z + s * d).cuda(), t)
        side.append(float((q.log_probs * w[0] + q.entropy * w[1] + q.lse * w[2]).sum()))
    slope, scale = (float((f(grad.cpu().double()) * f(d.double())).sum()) for f in (lambda x: x, torch.abs))
    assert abs((side[0] - side[1]) / (2 * h) - slope) < 2e-3 * scale


def test_rated(experts):  # noqa: F811
    z, t = scores(50, 700, "normal", torch.bfloat16, 4).cuda(), targets_of(50, 700, 4)
    plain = experts.rate(z, t, top_k=2)
    want = experts.rate_backward(z, t, plain, grad_log_probs=torch.full((50,), -0.5, device="cuda"), grad_entropy=torch.full((50,), 0.25, device="cuda"))
    z.requires_grad_()
    r = experts.rated(z, t, top_k=2)
    for a, b in zip(r, plain):
        assert torch.equal(a, b)
    loss = -0.5 * r.log_probs.sum() + 0.25 * r.entropy.sum()
    with torch.no_grad():
        r.top.add_(1)
        r.lse_rest.zero_()
    loss.backward()
    assert torch.equal(z.grad, want)
    # results changed in place leave the gradient as it is
    z.grad = None
    r = experts.rated(z, t)
    r.log_probs.mul_(-0.5)
    r.entropy.mul_(0.25)
    (r.log_probs.sum() + r.entropy.sum()).backward()
    assert torch.equal(z.grad, want)
    with torch.no_grad():
        assert not experts.rated(z, t).log_probs.requires_grad


# ---- dropout ----


def check_drop(experts, x, p, key, site, base, dtype):  # noqa: F811
    n, d = x.shape
    seed, step = (int(v) for v in key.tolist())
    keep = (ref.words(n * d, seed, step, site) >= min(round(p * 2**32), 2**32 - 1)).reshape(n, d)
    b = f64(base) if base is not None else np.zeros((n, d))
    want = np.where(keep, f64(x), 0.0) / (1 - p) + b
    bound = 4 * U * (np.abs(want) + np.abs(want - b)) + HALF[dtype] * np.abs(want) + STEP[dtype]
    out = experts.drop(x, p, key, site=site, base=base)
    near(out, want, bound, "out")
    assert out.dtype == x.dtype and out.is_contiguous()
    return out, keep


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,p", [(1, 1, 0.5), (1, 1000, 0.1), (3, 5, 0.25), (64, 128, 0.1), (33, 36, 0.9), (7, 1001, 0.0), (300, 24, 0.5), (5, 4, 1 - 2.0**-40)])
def test_drop(experts, n, d, p, dtype):  # noqa: F811
    print("drop", n, d, p, dtype, flush=True)
    g = torch.Generator().manual_seed(n + d)
    x, base = (torch.randn(n, d, generator=g).to(TYPES[dtype]).cuda() for _ in range(2))
    key = torch.tensor([-(2**62) + 12345, 2**35 + 7], device="cuda")
    for site in (0, 2**32 - 1):
        for b in (None, base):
            if p < 0.99 or dtype == "fp32":
                check_drop(experts, x, p, key, site, b, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [8, 12, 13, 64, 65])
def test_drop_places(experts, d, dtype):  # noqa: F811
    """The mask goes by the element's place, however its rows lie; out in x's or base's place."""
    g = torch.Generator().manual_seed(d)
    n, t = 41, TYPES[dtype]
    key = torch.tensor([99, 3], device="cuda")
    wide, more = (torch.randn(n, 100, generator=g).to(t).cuda() for _ in range(2))
    x, base = wide[:, 3 : 3 + d], more[:, 7 : 7 + d]
    want, keep = check_drop(experts, x, 0.3, key, 5, base, dtype)
    assert torch.equal(want, experts.drop(x.contiguous(), 0.3, key, site=5, base=base.contiguous()))
    assert torch.equal(want, experts.drop(x.contiguous(), 0.3, key, site=5, base=base))
    for place, opt in ((wide.clone(), "x"), (more.clone(), "base")):
        kept = place.clone()
        at = slice(3, 3 + d) if opt == "x" else slice(7, 7 + d)
        view = place[:, at]
        got = experts.drop(view if opt == "x" else x, 0.3, key, site=5, base=view if opt == "base" else base, out=view)
        assert torch.equal(got, want)
        kept[:, at] = want
        assert torch.equal(place, kept)
    x = torch.where(torch.from_numpy(keep).cuda(), x, math.nan)  # a dropped element does not reach out
    assert torch.equal(want, experts.drop(x, 0.3, key, site=5, base=base))
    one = wide[:1, :d].expand(n, d)
    check_drop(experts, one, 0.3, key, 5, one, dtype)


def test_drop_large_place(experts):  # noqa: F811
    """More than 2^32 elements: the counter's upper half, places past 32 bits."""
    n, d = 2**17 + 1, 2**15
    x = torch.ones(n, d, dtype=torch.bfloat16, device="cuda")
    key = torch.tensor([7, 9], device="cuda")
    out = experts.drop(x, 0.5, key, out=x)
    counter = n * d // 4 - 64  # the last 256 elements
    got = out.view(-1)[-256:].cpu()
    c = []
    for b in range(counter, counter + 64):
        w = [b & 0xFFFFFFFF, b >> 32, 0, 9]
        k0, k1 = 7, 0
        for _ in range(10):
            p, q = 0xD2511F53 * w[0], 0xCD9E8D57 * w[2]
            w = [(q >> 32) ^ w[1] ^ k0, q & 0xFFFFFFFF, (p >> 32) ^ w[3] ^ k1, p & 0xFFFFFFFF]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        c += w
    assert counter > 2**30 and got.tolist() == [2.0 if v >= 2**31 else 0.0 for v in c]


def test_dropped(experts):  # noqa: F811
    key = torch.tensor([5, 1], device="cuda")
    x, base = (torch.randn(30, 48, device="cuda", requires_grad=True) for _ in range(2))
    dy = torch.randn(30, 48, device="cuda")
    y = experts.dropped(x, 0.4, key, site=2, base=base)
    assert torch.equal(y, experts.drop(x.detach(), 0.4, key, site=2, base=base.detach()))
    y.backward(dy)
    assert torch.equal(base.grad, dy) and torch.equal(x.grad, experts.drop(dy, 0.4, key, site=2))
    x.grad = None
    experts.dropped(x, 0.4, key).sum().backward()  # a gradient of one value for all elements
    assert torch.equal(x.grad, experts.drop(torch.ones(30, 48, device="cuda"), 0.4, key))
    y = experts.dropped(x, 0.4, key)
    key[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert not torch.equal(experts.drop(dy, 0.4, key), experts.drop(dy, 0.4, torch.tensor([5, 1], device="cuda")))


def test_python_refusals(experts):  # noqa: F811
    x, key = torch.zeros(4, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for p in (-0.1, 1.0, math.nan):
        with pytest.raises(ValueError, match="p="):
            experts.drop(x, p, key)
    with pytest.raises(ValueError, match="site="):
        experts.drop(x, 0.1, key, site=1 << 32)
    with pytest.raises(TypeError, match="key"):
        experts.drop(x, 0.1, key.int())
    with pytest.raises(ValueError, match="key"):
        experts.drop(x, 0.1, key[:1])
    with pytest.raises(ValueError, match="on cpu"):
        experts.drop(x, 0.1, key.cpu())
    with pytest.raises(ValueError, match="base"):
        experts.drop(x, 0.1, key, base=x[:3])
    wide = torch.zeros(4, 20, device="cuda")
    with pytest.raises(RuntimeError, match="out shares memory with x"):
        experts.drop(wide[:, :8], 0.1, key, out=wide[:, 1:9])
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="top_k"):
        experts.rate(x, t, top_k=9)
    with pytest.raises(TypeError, match="targets"):
        experts.rate(x, t.long())
    with pytest.raises(ValueError, match="targets"):
        experts.rate(x, t[:3])
    with pytest.raises(ValueError, match="side by side"):
        experts.rate(x.T, torch.zeros(8, dtype=torch.int32, device="cuda"))
    r = experts.rate(x, t)
    with pytest.raises(ValueError, match="grad_entropy"):
        experts.rate_backward(x, t, r, grad_entropy=torch.zeros(3, device="cuda"))
