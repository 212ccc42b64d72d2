"""Which way the feed-forward takes few slots, by the workspace that it asks for: without a sort only the hidden vectors'."""

from __future__ import annotations

import pytest


def few(dtype, n, d, f, o, k, a):
    """Whether no way that a call may take its rows and matrices has a sort."""
    from skmetal_amd import _bridge

    if _bridge._lib is None:
        pytest.fail(f"library not loaded: {_bridge.last_error()}")
    vec = 4 if dtype == 0 else 8
    return _bridge._lib.skmetal_hip_feed_workspace(dtype, n, d, f, o, k, a, 0) == n * k * -(-f // vec) * 16


@pytest.mark.parametrize("dtype,n,d,f,k,a", [
    (1, 1, 2048, 1024, 2, 8), (1, 1, 4096, 11_008, 1, 1), (1, 4, 4096, 11_008, 1, 1), (2, 8, 4096, 2048, 1, 1), (1, 16, 512, 512, 4, 64), (1, 8, 2048, 1024, 2, 8), (0, 1, 4096, 2048, 2, 8),
    (0, 12, 4096, 2048, 1, 1), (0, 48, 512, 512, 1, 1), (0, 48, 1024, 1024, 1, 1), (1, 1, 16_384, 53_248, 1, 1),
])
def test_a_few_slots_go_without_a_sort(dtype, n, d, f, k, a):
    assert few(dtype, n, d, f, d, k, a)


@pytest.mark.parametrize("dtype,n,d,f,k,a", [
    (1, 16, 4096, 11_008, 1, 1), (1, 12, 4096, 11_008, 1, 2), (1, 16, 4096, 2048, 1, 2), (2, 8, 4096, 2048, 2, 4), (1, 32, 2048, 1024, 1, 1), (0, 48, 4096, 2048, 1, 1),
    (0, 48, 4096, 11_008, 1, 1), (0, 16, 4096, 2048, 2, 4), (1, 65, 512, 512, 1, 64), (1, 16, 16_384, 53_248, 1, 1),
])
def test_slots_that_share_experts_read_a_matrix_once(dtype, n, d, f, k, a):
    """Reading it once a slot took up to 5.8 times as long as tiles (48 rows of one fp32 block of 4,096 by 11,008)."""
    assert not few(dtype, n, d, f, d, k, a)
