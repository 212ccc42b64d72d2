"""The routing and adapter operators without a GPU: their references' gradients against
differences, and the refusals of the C entry points (arguments are checked before the
device)."""

from __future__ import annotations

import ctypes

import experts_reference as ref
import numpy as np
import pytest

EINVAL, ENODEV, ERANGE = 1, 2, 6


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("excluded", [False, True])
def test_route_reference_gradient_is_its_difference(normalize, excluded):
    rng = np.random.default_rng(11)
    n, e, k = 9, 7, 3
    z = rng.standard_normal((n, e)) * 2
    if excluded:
        z[rng.random((n, e)) < 0.2] = -np.inf
        z[4] = -np.inf
    mask = np.ones(n, bool)
    mask[2] = False
    dw, dl = rng.standard_normal((n, k)), 1.7
    w, ex, counts, _, rows, _, p = ref.route(z, k, mask, normalize)
    got, _ = ref.route_backward(p, w, ex, counts, rows, dw, dl, normalize)

    def value(zz):
        w2, ex2, c2, sums, r2, loss, _ = ref.route(zz, k, mask, normalize)
        assert (ex2 == ex).all() and (c2 == counts).all() and r2 == rows
        return float((w2 * dw).sum()) + dl * loss

    h = 1e-6  # central differences: h^2 truncation and 2^-53 / h rounding, both under 1e-9 here
    for i in range(n):
        for j in range(e):
            if not np.isfinite(z[i, j]):
                assert got[i, j] == 0
                continue
            up, dn = z.copy(), z.copy()
            up[i, j] += h
            dn[i, j] -= h
            assert abs((value(up) - value(dn)) / (2 * h) - got[i, j]) < 1e-8


def test_adapt_reference_gradient_is_its_difference():
    rng = np.random.default_rng(12)
    n, d, o, r, a = 6, 5, 4, 2, 3
    x, A, B = rng.standard_normal((n, d)), rng.standard_normal((a, r, d)), rng.standard_normal((a, r, o))
    ids, gates, scales = np.array([0, 2, 2, -1, 0, 5]), rng.random(n), rng.random(a) + 0.5
    dy = rng.standard_normal((n, o))
    (dx, dA, dB, dg), _ = ref.adapt_backward(dy, x, A, B, ids, None, gates, scales)

    def value():
        return float((ref.adapt(x, A, B, ids, None, gates, scales)[0] * dy).sum())

    h = 1e-6
    for v, g in ((x, dx), (A, dA), (B, dB), (gates, dg)):
        flat, gf = v.reshape(-1), g.reshape(-1)
        for i in range(flat.size):
            keep = flat[i]
            flat[i] = keep + h
            hi = value()
            flat[i] = keep - h
            lo = value()
            flat[i] = keep
            assert abs((hi - lo) / (2 * h) - gf[i]) < 1e-8


@pytest.fixture(scope="module")
def lib():
    from skmetal_amd import _bridge

    if _bridge._lib is None:
        pytest.fail(f"library not loaded: {_bridge.last_error()}")
    return _bridge._lib


P = 4096  # a pointer that no call below gets to use


def _route(lib, dtype=1, z=P, ld=64, mask=None, n=8, e=64, k=2, w=P, ex=P, c=P, s=P, rows=P, loss=P, ws=P, size=1 << 30):
    return lib.skmetal_hip_route(dtype, z, ld, mask, 1, n, e, k, 0, w, ex, c, s, rows, loss, ws, size, None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(dtype=3), EINVAL, "dtype"), (dict(k=0), EINVAL, "k=0"), (dict(k=65), EINVAL, "k=65"), (dict(e=0, k=0), EINVAL, "E=0"),
    (dict(e=4096, k=2), ERANGE, "E=4096"), (dict(k=17), ERANGE, "k=17"), (dict(n=1 << 31), ERANGE, "n="), (dict(ld=1 << 50), ERANGE, "stride"),
    (dict(z=None), EINVAL, "null"), (dict(w=None), EINVAL, "null"), (dict(loss=None), EINVAL, "null"), (dict(z=P + 1), EINVAL, "aligned"),
    (dict(n=100_000, size=16), EINVAL, "workspace"), (dict(n=100_000, ws=None), EINVAL, "workspace"), (dict(n=100_000, ws=P + 4), EINVAL, "aligned"),
])
def test_route_refuses(lib, bad, code, says):
    assert _route(lib, **bad) == code
    assert says in lib.skmetal_hip_last_error().decode()


def _adapt(lib, dtype=1, x=P, down=P, up=P, ids=P, base=P, out=P, ld_out=64, n=8, d=64, o=64, r=8, a=4, ws=P, size=1 << 40):
    return lib.skmetal_hip_adapt(dtype, x, d, down, r * d, d, up, r * o, o, ids, 1, None, 0, None, base, o, out, ld_out, None, n, d, o, r, a, ws, size, None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(dtype=-1), EINVAL, "dtype"), (dict(r=0), EINVAL, "r=0"), (dict(d=0), EINVAL, "d=0"), (dict(r=129), ERANGE, "r=129"), (dict(a=65536), ERANGE, "a=65536"),
    (dict(n=1 << 31), ERANGE, "n="), (dict(x=None), EINVAL, "null"), (dict(up=None), EINVAL, "null"), (dict(ids=None), EINVAL, "null"),
    (dict(out=P + 1), EINVAL, "aligned"), (dict(ld_out=63), EINVAL, "overlap"), (dict(n=1 << 29, d=1 << 20), ERANGE, "blocks"),
])
def test_adapt_refuses(lib, bad, code, says):
    assert _adapt(lib, **bad) == code
    assert says in lib.skmetal_hip_last_error().decode()


def test_backward_refuses(lib):
    def route_back(k=2, ex=P, grad=P, ld=64):
        return lib.skmetal_hip_route_backward(1, P, 64, None, 0, 8, 64, k, 0, P, ex, P, P, None, None, grad, ld, None)

    def adapt_back(r=8, low=P, dA=P, ld=64, size=1 << 40):
        return lib.skmetal_hip_adapt_backward(1, P, 64, P, 64, P, 512, 64, P, 512, 64, P, 1, None, 0, None, low, None, 0, P, ld, dA, P, None, 8, 64, 64, r, 4, P,
                                              size, None)

    for call, bad, code in ((route_back, dict(k=99), EINVAL), (route_back, dict(ex=None), EINVAL), (route_back, dict(grad=P + 1), EINVAL),
                            (route_back, dict(ld=63), EINVAL), (adapt_back, dict(r=500), ERANGE), (adapt_back, dict(low=None), EINVAL),
                            (adapt_back, dict(dA=None), EINVAL), (adapt_back, dict(ld=1), EINVAL), (adapt_back, dict(size=0), EINVAL)):
        assert call(**bad) == code, bad


def test_a_call_without_a_device_says_so(lib):
    from skmetal_amd import _bridge

    if _bridge.HIP_AVAILABLE:
        pytest.skip("a GPU is present")
    assert _route(lib) == ENODEV and _adapt(lib) == ENODEV
    assert "skmetal_init" in lib.skmetal_hip_last_error().decode()


def test_tensors_that_are_not_on_the_gpu_are_refused():
    torch = pytest.importorskip("torch")
    from skmetal_amd import experts

    with pytest.raises(ValueError, match="expected the GPU"):
        experts.route(torch.zeros(4, 8), 2)
    with pytest.raises(TypeError, match="float64"):
        experts.route(torch.zeros(4, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="expected the GPU"):
        experts.adapt(torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.zeros(1, 2, 8), torch.zeros(4, dtype=torch.int32))


def test_workspace_sizes_cover_every_call_they_are_asked_for(lib):
    assert lib.skmetal_hip_route_workspace(1 << 40, 8) == 0 and lib.skmetal_hip_adapt_workspace(7, 8, 8, 8, 8, 8, 0) == 0
    assert ctypes.c_size_t(lib.skmetal_hip_route_workspace(100_000, 2048)).value < 1 << 30


@pytest.mark.parametrize("first", ["torch", "skmetal_amd"])
def test_torch_and_the_library_share_one_runtime(first):
    """Whichever of the two is imported first."""
    import subprocess
    import sys
    from pathlib import Path

    torch = pytest.importorskip("torch")
    if not (Path(torch.__file__).parent / "lib" / "libamdhip64.so").exists():
        pytest.skip("this torch brings no HIP runtime")
    code = f"import {first}\nimport skmetal_amd, torch\nfrom skmetal_amd import _bridge\n_bridge.require_torch_runtime()"
    done = subprocess.run([sys.executable, "-W", "ignore", "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
