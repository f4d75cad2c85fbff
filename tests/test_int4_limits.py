"""Sizes of the 4-bit linear that no launch holds, on the host: refused, whatever they come to in 32 bits."""

from __future__ import annotations

import ctypes

import pytest

from flextensor_amd import _native as nat


@pytest.mark.parametrize("m,n", [
    (1 << 40, 1), ((1 << 38) + 320, 1), ((1 << 38) - 1, 1), (1 << 38, 1), ((1 << 38) - 11 * 64, 1), (1 << 37, 2), (1 << 33, 100),
    ((1 << 40) - 1, 1), (1 << 36, 16), (33, 1 << 34), (1 << 20, 1 << 20),
])
@pytest.mark.parametrize("k,group", [(128, 128), (32, 32), (1 << 20, 64)])
def test_more_rows_or_channels_than_a_launch_holds_are_refused(m, n, k, group):
    b = ctypes.c_size_t(7)
    lib = nat.load()
    assert lib.ftx_int4_linear_workspace(m, n, k, group, ctypes.byref(b)) == nat.FTX_ERR_UNSUPPORTED and b.value == 7
    # the shape is looked at before any pointer
    assert lib.ftx_int4_linear(None, k, None, None, None, None, m, n, k, group, None, 0, None) == nat.FTX_ERR_UNSUPPORTED


@pytest.mark.parametrize("m,n,k", [(1 << 24, 128, 128), ((1 << 24) + 63, 1, 64), (17, 1 << 24, 32)])
def test_the_largest_sizes_have_a_plan(m, n, k):
    b = ctypes.c_size_t(7)
    assert nat.load().ftx_int4_linear_workspace(m, n, k, 32, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
