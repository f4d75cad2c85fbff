"""The 4-bit linear of 17 to 32 rows, two tiles of rows at once: weights enter the products exactly, so a result is off
by its own rounding to bf16, half a step or 2^-8 of itself, and by fp32 sums, 2^-24 of 16 times the terms for each of the
k / 32 steps of a sum.
"""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import hip

pytestmark = pytest.mark.gpu


def _weights(gpu, n, k, group, zeros, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), device=gpu, generator=g)
    scale = (torch.rand(n, k // group, device=gpu, generator=g) * 0.02 + 0.001).bfloat16()
    zero = (torch.rand(n, k // group, device=gpu, generator=g) * 15).bfloat16() if zeros else None
    return hip.int4_pack(codes, scale, zero)


@pytest.mark.parametrize("group,zeros", [(128, False), (128, True), (64, False), (64, True), (32, False), (32, True)])
@pytest.mark.parametrize("m,n,k", [(17, 16, 128), (18, 1, 384), (25, 300, 512), (31, 4100, 640), (32, 4096, 1024),
                                   (32, 9000, 256), (29, 17, 4096)])
def test_rows_of_two_tiles_are_the_definition(gpu, m, n, k, group, zeros):
    packed = _weights(gpu, n, k, group, zeros)
    x = torch.randn(m, k, device=gpu, generator=torch.Generator(device=gpu).manual_seed(m)).bfloat16()
    w = hip.int4_dequantize(*packed, n, k).double()
    want, terms = x.double() @ w.T, x.double().abs() @ w.abs().T
    got = hip.int4_linear(x, *packed, n=n).double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 16 * (k / 32) * 2.0 ** -24 * terms + 1e-30).all()
    for i in (0, 15, 16, m - 1):  # a row's result does not depend on the others
        assert torch.equal(hip.int4_linear(x.roll(-i, 0), *packed, n=n).double().roll(i, 0), got)


def test_rows_apart_and_of_odd_groups(gpu):
    """Strided rows, and a k that ends inside a unit."""
    for k, group in ((32, 32), (96, 32), (192, 64), (1000 // 32 * 32, 32)):
        packed = _weights(gpu, 70, k, group, True, 1)
        wide = torch.randn(32, k + 24, device=gpu, generator=torch.Generator(device=gpu).manual_seed(k)).bfloat16()
        got = hip.int4_linear(wide[:, :k], *packed, n=70)
        assert torch.equal(got, hip.int4_linear(wide[:, :k].contiguous(), *packed, n=70))
        want = wide[:, :k].double() @ hip.int4_dequantize(*packed, 70, k).double().T
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_a_row_that_is_not_finite_leaves_the_others_alone(gpu):
    packed = _weights(gpu, 200, 256, 64, True, 2)
    x = torch.randn(30, 256, device=gpu, generator=torch.Generator(device=gpu).manual_seed(0)).bfloat16()
    want = hip.int4_linear(x, *packed, n=200)
    x[3, 7], x[20, 200] = float("inf"), float("nan")
    got = hip.int4_linear(x, *packed, n=200)
    rest = [i for i in range(30) if i not in (3, 20)]
    assert torch.equal(got[rest], want[rest]) and not got[[3, 20]].isfinite().any()


def test_replays_of_a_captured_call(gpu):
    packed = _weights(gpu, 3000, 512, 128, False, 3)
    x = torch.zeros(27, 512, device=gpu).bfloat16()
    hip.int4_linear(x, *packed, n=3000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip.int4_linear(x, *packed, n=3000)
    for seed in range(4):
        x.copy_(torch.randn(27, 512, device=gpu, generator=torch.Generator(device=gpu).manual_seed(seed)))
        graph.replay()
        assert torch.equal(out, hip.int4_linear(x, *packed, n=3000))
