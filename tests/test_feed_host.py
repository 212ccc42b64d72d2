"""The feed-forward, dropout and log-probability operators without a GPU: the refusals of the C entry points
(arguments are checked before the device), what the Python calls hand to the library, and workspaces."""

from __future__ import annotations

import types

import pytest

EINVAL, ENODEV, ERANGE = 1, 2, 6
P = 1 << 20  # addresses that no call below gets to use


@pytest.fixture(scope="module")
def lib():
    from skmetal_amd import _bridge

    if _bridge._lib is None:
        pytest.fail(f"library not loaded: {_bridge.last_error()}")
    if _bridge.HIP_AVAILABLE:
        pytest.skip("an accepted call would run on these addresses")
    return _bridge._lib


def _feed(lib, dtype=1, x=P, gate=2 * P, up=3 * P, down=4 * P, chosen=5 * P, weights=6 * P, act=0, base=7 * P, ld_base=64, out=8 * P, ld_out=64, pre=None, n=8, d=64, f=32,
          o=64, k=2, a=4, ws=9 * P, size=1 << 40, ld_x=64, ld_gate=64):
    return lib.skmetal_hip_feed(dtype, x, ld_x, gate, f * d, ld_gate, up, f * d, d, down, o * f, f, chosen, weights, act, base, ld_base, out, ld_out, pre, n, d, f, o, k, a,
                                ws, size, None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(dtype=3), EINVAL, "dtype"), (dict(d=0), EINVAL, "d=0"), (dict(f=0), EINVAL, "f=0"), (dict(o=0), EINVAL, "o=0"), (dict(k=0), EINVAL, "k=0"), (dict(a=0), EINVAL, "a=0"),
    (dict(act=3), EINVAL, "act=3"), (dict(k=17), ERANGE, "k=17"), (dict(a=2049), ERANGE, "a=2049"), (dict(n=1 << 30), ERANGE, "n="), (dict(n=1 << 29, k=4), ERANGE, "blocks"),
    (dict(ld_x=1 << 50), ERANGE, "stride"), (dict(ld_gate=1 << 50), ERANGE, "stride"), (dict(x=None), EINVAL, "null"), (dict(gate=None), EINVAL, "null"),
    (dict(down=None), EINVAL, "null"), (dict(out=None), EINVAL, "null"), (dict(chosen=None), EINVAL, "chosen is null"), (dict(chosen=None, k=1), EINVAL, "chosen is null"),
    (dict(x=P + 1), EINVAL, "aligned"), (dict(up=P + 1), EINVAL, "aligned"), (dict(out=8 * P + 1), EINVAL, "aligned"), (dict(ld_out=63), EINVAL, "overlap"),
    (dict(base=8 * P + 2), EINVAL, "out shares memory with base"), (dict(base=8 * P, ld_base=128), EINVAL, "out shares memory with base"),
    (dict(size=16), EINVAL, "workspace"), (dict(ws=None), EINVAL, "workspace"), (dict(ws=9 * P + 4), EINVAL, "aligned"),
])
def test_feed_refuses(lib, bad, code, says):
    assert _feed(lib, **bad) == code, lib.skmetal_hip_last_error()
    assert says in lib.skmetal_hip_last_error().decode()


def test_feed_accepts_large_models(lib):
    """Many experts of wide blocks, and many rows: the launches of both directions have room."""
    for z in (dict(n=4096, d=7168, f=2048, o=7168, k=8, a=256), dict(n=1 << 16, d=4096, f=14_336, o=4096, k=2, a=8), dict(n=1 << 20, d=2048, f=1024, o=2048, k=8, a=128),
              dict(n=1, d=16_384, f=53_248, o=16_384, k=1, a=1), dict(n=512, d=4096, f=4096, o=4096, k=4, a=2048)):
        for dtype in (0, 1, 2):
            assert all(lib.skmetal_hip_feed_workspace(dtype, *z.values(), b) > 0 for b in (0, 1)), (z, lib.skmetal_hip_last_error())
        big = dict(x=1 << 44, out=1 << 45, base=None, ld_x=z["d"], ld_gate=z["d"], ld_out=z["o"], size=1 << 50, **z)
        assert _feed(lib, **big) == ENODEV, lib.skmetal_hip_last_error()


def test_feed_accepts(lib):
    """Up to the missing device: in place, without a router, weights or base, no rows, x anywhere."""
    for good in (dict(), dict(base=8 * P), dict(base=None), dict(weights=None), dict(chosen=None, k=1, a=1), dict(n=0, x=None, out=None, chosen=None), dict(x=8 * P), dict(x=P + 2),
                 dict(n=1, ld_out=0), dict(ld_x=0)):
        assert _feed(lib, **good) == ENODEV, good


def _feed_back(lib, grad=P, x=2 * P, pre=3 * P, base=None, grad_x=4 * P, ld_grad_x=64, dm=(5 * P, 6 * P, 7 * P), dw=8 * P, n=8, d=64, f=32, o=64, k=2, a=4, act=1, chosen=9 * P,
               size=1 << 40):
    return lib.skmetal_hip_feed_backward(0, grad, o, x, d, P // 2, f * d, d, P // 2, f * d, d, P // 2, o * f, f, chosen, None, act, pre, base, 64, grad_x, ld_grad_x, *dm, dw, n, d, f,
                                         o, k, a, 10 * P, size, None)


@pytest.mark.parametrize("bad,says", [
    (dict(grad=None), "null"), (dict(pre=None), "null"), (dict(x=None), "null"), (dict(dm=(5 * P, 6 * P, None)), "together"), (dict(dm=(None, None, 7 * P)), "together"),
    (dict(act=-1), "act"), (dict(ld_grad_x=63), "overlap"), (dict(grad_x=P), "grad_x shares memory with grad or x"), (dict(grad_x=2 * P + 4 * 100), "grad_x shares memory with grad or x"),
    (dict(base=4 * P + 4), "grad_x shares memory with base"), (dict(size=0), "workspace"), (dict(dm=(5 * P + 1, 6 * P, 7 * P)), "aligned"), (dict(chosen=None), "chosen is null"),
])
def test_feed_backward_refuses(lib, bad, says):
    assert _feed_back(lib, **bad) == EINVAL
    assert says in lib.skmetal_hip_last_error().decode()


def test_feed_backward_accepts(lib):
    for good in (dict(), dict(grad_x=None), dict(dm=(None, None, None)), dict(dw=None), dict(base=4 * P), dict(n=0, grad=None, x=None, pre=None, chosen=None)):
        assert _feed_back(lib, **good) == ENODEV, good


def _drop(lib, dtype=1, x=P, ld_x=64, base=None, ld_base=64, out=2 * P, ld_out=64, n=8, d=64, p=0.1, key=3 * P):
    return lib.skmetal_hip_drop(dtype, x, ld_x, base, ld_base, out, ld_out, n, d, p, key, 7, None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(dtype=9), EINVAL, "dtype"), (dict(p=1.0), EINVAL, "p=1"), (dict(p=-0.5), EINVAL, "p=-0.5"), (dict(p=float("nan")), EINVAL, "p="), (dict(d=0), EINVAL, "d must"),
    (dict(n=1 << 31), ERANGE, "n="), (dict(ld_x=1 << 50), ERANGE, "stride"), (dict(key=None), EINVAL, "null"), (dict(x=None), EINVAL, "null"), (dict(out=None), EINVAL, "null"),
    (dict(ld_out=63), EINVAL, "overlap"), (dict(key=3 * P + 4), EINVAL, "key is not aligned"), (dict(out=2 * P + 1), EINVAL, "aligned"), (dict(out=P + 2), EINVAL, "out shares memory with x"),
    (dict(out=P, ld_out=128), EINVAL, "out shares memory with x"), (dict(base=2 * P + 2), EINVAL, "out shares memory with base"), (dict(key=2 * P + 8), EINVAL, "out shares memory with key"),
])
def test_drop_refuses(lib, bad, code, says):
    assert _drop(lib, **bad) == code
    assert says in lib.skmetal_hip_last_error().decode()


def test_drop_accepts(lib):
    for good in (dict(), dict(out=P), dict(base=2 * P), dict(base=P, out=P), dict(n=0, x=None, out=None), dict(p=0.0), dict(x=P, ld_x=128, out=P + 128, ld_out=128), dict(ld_x=0)):
        assert _drop(lib, **good) == ENODEV, good


def _rate(lib, dtype=1, z=P, ld=100, t=2 * P, n=8, v=100, k=4, lp=3 * P, top=4 * P, ws=5 * P, size=1 << 30):
    return lib.skmetal_hip_rate(dtype, z, ld, t, 1, n, v, k, lp, lp, lp, lp, top, top, ws, size, None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(dtype=-1), EINVAL, "dtype"), (dict(v=0, k=0), EINVAL, "v=0"), (dict(k=101), EINVAL, "k=101"), (dict(k=17), ERANGE, "k=17"), (dict(v=(1 << 22) + 1), ERANGE, "scores a row"),
    (dict(n=1 << 31), ERANGE, "n="), (dict(n=1 << 24, v=1 << 22), ERANGE, "blocks"), (dict(ld=1 << 50), ERANGE, "stride"), (dict(z=None), EINVAL, "null"), (dict(t=None), EINVAL, "null"),
    (dict(lp=None), EINVAL, "null"), (dict(top=None), EINVAL, "null"), (dict(z=P + 1), EINVAL, "aligned"), (dict(v=1 << 20, size=8), EINVAL, "workspace"),
    (dict(v=1 << 20, ws=None), EINVAL, "workspace"),
])
def test_rate_refuses(lib, bad, code, says):
    assert _rate(lib, **bad) == code
    assert says in lib.skmetal_hip_last_error().decode()


def test_rate_accepts(lib):
    for good in (dict(), dict(k=0, top=None), dict(n=0, z=None, t=None, lp=None, top=None), dict(v=1 << 22, k=16), dict(ws=None, size=0)):
        assert _rate(lib, **good) == ENODEV, good

    def back(z=P, ld=100, dz=2 * P, ld_dz=100, lse=3 * P):
        return lib.skmetal_hip_rate_backward(0, z, ld, 4 * P, 1, 8, 100, lse, lse, lse, None, None, None, dz, ld_dz, None)

    assert back() == ENODEV and back(dz=P) == ENODEV
    for bad in (dict(dz=None), dict(lse=None), dict(ld_dz=99), dict(dz=P + 4), dict(dz=P, ld_dz=101)):
        assert back(**bad) == EINVAL, bad


def test_workspaces(lib):
    assert lib.skmetal_hip_feed_workspace(1, 8, 0, 32, 64, 2, 4, 0) == 0 and lib.skmetal_hip_rate_workspace(1, 1 << 40, 8, 2) == 0
    assert lib.skmetal_hip_rate_workspace(1, 5000, 32_000, 0) == 0 and lib.skmetal_hip_rate_workspace(1, 1, 1 << 22, 16) < 1 << 20


@pytest.mark.parametrize("n,d,f,o,k,a", [(8192, 2048, 2048, 2048, 2, 8), (64, 4096, 2048, 4096, 2, 16), (4096, 2048, 8192, 2048, 1, 1), (16, 512, 512, 512, 16, 2048), (1000, 777, 501, 33, 3, 5)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces_follow_the_slots(lib, n, d, f, o, k, a, dtype):
    """h (and its gradients) a slot, fp32 results a slot in at most 4 parts, a few numbers a slot and an expert; the
    matrices' gradients in fp32 parts only where there are few tiles of them (at most 512 blocks' worth)."""
    es = 4 if dtype == 0 else 2
    slots = n * k
    few = 16 * slots + 64 * (a + 1) + 8 * (a + 1) * (slots // 16_384 + 1) + 2048
    forward, backward = (lib.skmetal_hip_feed_workspace(dtype, n, d, f, o, k, a, b) for b in (0, 1))
    assert 0 < forward <= slots * (f + 8) * es + 16 * slots * o + few
    assert 0 < backward <= 3 * slots * (f + 8) * es + 8 * slots * d + 4 * slots * (f // 32 + 2) + 512 * 256 * 256 * 4 + few


# ---- what the Python calls hand over ----


@pytest.fixture
def calls(monkeypatch):
    """Calls that reached the library, as (entry point, arguments)."""
    torch = pytest.importorskip("torch")  # noqa: F841
    from skmetal_amd import experts

    made = []

    def entry(name):
        return lambda *args: made.append((name, args)) or 0

    names = ("feed", "feed_backward", "drop", "rate", "rate_backward")
    monkeypatch.setattr(experts, "_lib", lambda: types.SimpleNamespace(**{f"skmetal_hip_{n}": entry(n) for n in names}))
    monkeypatch.setattr(experts, "_first", lambda t, name: (experts._CODE[t.dtype], t.device))
    monkeypatch.setattr(experts, "_stream", lambda device: None)
    monkeypatch.setattr(experts, "_feed_workspace", lambda *sizes: 0)
    monkeypatch.setattr(experts, "_rate_workspace", lambda *sizes: 0)
    return made


def test_strides_as_they_are(calls):
    import torch
    from skmetal_amd import experts

    both = torch.zeros(3, 96, 40)  # gate and up as halves of one tensor
    x, chosen = torch.zeros(10, 50)[:, 3:43], torch.zeros(10, 2, dtype=torch.int32)
    down = torch.zeros(3, 24, 60)[:, :, :48]
    out, pre = experts.feed(x, both[:, :48], both[:, 48:], down, chosen, base=torch.zeros(10, 30)[:, :24], act="gelu", return_pre=True)
    (name, args), = calls
    assert name == "feed" and out.shape == (10, 24) and pre.shape == (10, 2, 2, 48)
    assert args[2] == 50 and args[4:6] == (96 * 40, 40) and args[7:9] == (96 * 40, 40) and args[10:12] == (24 * 60, 60)
    assert args[13] is None and args[14] == 1 and args[16] == 30 and args[18] == 24 and args[20:26] == (10, 40, 48, 24, 2, 3)
    calls.clear()
    experts.feed_backward(torch.zeros(10, 70)[:, :24], x, both[:, :48], both[:, 48:], down, chosen, pre, rows=False)
    (name, args), = calls
    assert name == "feed_backward" and args[2] == 70 and args[20] is None and all(args[22:25]) and args[25] is None


def test_rows_whose_elements_lie_apart_are_refused(calls):
    import torch
    from skmetal_amd import experts

    apart = torch.zeros(16, 10).T
    m = torch.zeros(2, 8, 16), torch.zeros(2, 8, 16), torch.zeros(2, 16, 8)
    chosen, key, t = torch.zeros(10, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(10, dtype=torch.int32)
    for call in (lambda: experts.feed(apart, *m, chosen), lambda: experts.feed(torch.zeros(10, 16), *m, chosen, base=apart), lambda: experts.feed(torch.zeros(10, 16), *m, chosen, out=apart),
                 lambda: experts.drop(apart, 0.1, key), lambda: experts.drop(torch.zeros(10, 16), 0.1, key, base=apart), lambda: experts.rate(apart, t),
                 lambda: experts.feed(torch.zeros(10, 16), m[0], m[1].transpose(1, 2).contiguous().transpose(1, 2), m[2], chosen)):
        with pytest.raises(ValueError, match="side by side"):
            call()
    assert not calls


def test_out_is_known_to_autograd(calls):
    import torch
    from skmetal_amd import experts

    m = torch.zeros(1, 8, 16), torch.zeros(1, 8, 16), torch.zeros(1, 16, 8)
    key = torch.zeros(2, dtype=torch.int64)
    for call in (lambda y: experts.feed(y, *m, base=y, out=y), lambda y: experts.drop(y, 0.1, key, out=y)):
        w = torch.ones(16, requires_grad=True)
        y = torch.zeros(10, 16)
        z = y * w
        call(y)
        with pytest.raises(RuntimeError, match="inplace operation"):
            z.sum().backward()
        y = torch.zeros(10, 16) * w
        with pytest.raises(ValueError, match="out requires a gradient"):
            call(y)
        with torch.no_grad():
            call(y)


def test_fed_asks_for_what_is_needed(calls):
    """Frozen matrices, or rows that need no gradient, cost no product of theirs."""
    import torch
    from skmetal_amd import experts

    for need, rows, matrices in (((1, 0, 0), True, False), ((0, 1, 0), False, True), ((0, 0, 1), False, False), ((1, 1, 1), True, True)):
        x, w = torch.zeros(10, 16, requires_grad=bool(need[0])), torch.zeros(10, 1, requires_grad=bool(need[2]))
        gate, up = torch.zeros(2, 8, 16, requires_grad=bool(need[1])), torch.zeros(2, 8, 16)
        experts.fed(x, gate, up, torch.zeros(2, 16, 8), torch.zeros(10, 1, dtype=torch.int32), weights=w).sum().backward()
        name, args = calls[-1]
        assert name == "feed_backward" and (args[20] is not None) == rows and (args[22] is not None) == matrices
        assert (x.grad is not None, gate.grad is not None, w.grad is not None) == tuple(map(bool, need)) and up.grad is None
    calls.clear()
    base = torch.zeros(10, 16, requires_grad=True)  # the residual stream alone
    experts.fed(torch.zeros(10, 16), torch.zeros(1, 8, 16), torch.zeros(1, 8, 16), torch.zeros(1, 16, 8), base=base).sum().backward()
    assert [c[0] for c in calls] == ["feed"] and (base.grad == 1).all()


def test_without_the_gpu_the_calls_say_so():
    torch = pytest.importorskip("torch")
    from skmetal_amd import experts

    x, key = torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: experts.feed(x, torch.zeros(1, 4, 8), torch.zeros(1, 4, 8), torch.zeros(1, 8, 4)), lambda: experts.drop(x, 0.1, key),
                 lambda: experts.rate(x, torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError, match="expected the GPU"):
            call()
    with pytest.raises(TypeError, match="float64"):
        experts.rate(x.double(), torch.zeros(4, dtype=torch.int32))
