"""The 4-bit linear against float64 over the weights that its codes stand for.

Up to 16 rows an output is rounded once: half a step of bf16, 2^-8 of the value, and what fp32 sums lose of numbers up
to 151 = 128 + 15 + 8 times a scale, 2^-24 of them for each of the 128 + 8 additions within a group and behind it. More
rows round each weight to bf16 as well: another 2^-8 of |x| |w| at most, and 2^-24 of it for each addition.
"""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import hip

pytestmark = pytest.mark.gpu

ONE_ROUNDING = 2.0 ** -8
TWO_ROUNDINGS = 2.0 ** -7


def _inputs(gpu, m, n, k, group, zeros, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + m + 3 * n + 7 * k + group)
    x = torch.randn(m, k, device=gpu, generator=g)
    x[:, :: max(1, k // 8)] *= 8.0
    codes = torch.randint(0, 16, (n, k), device=gpu, generator=g, dtype=torch.int32)
    scale = (torch.exp(0.2 * torch.randn(n, k // group, device=gpu, generator=g)) * 1e-2).bfloat16()
    zero = (8 + 3 * torch.randn(n, k // group, device=gpu, generator=g)).bfloat16() if zeros else None
    return x.bfloat16(), codes, scale, zero


def _weights(codes, scale, zero):
    group = codes.shape[1] // scale.shape[1]
    z = zero.double() if zero is not None else torch.full_like(scale, 8.0, dtype=torch.float64)
    return (codes.double() - z.repeat_interleave(group, 1)) * scale.double().repeat_interleave(group, 1)


def _check(y, x, codes, scale, zero):
    w = _weights(codes, scale, zero)
    exact = x.double() @ w.t()
    group = codes.shape[1] // scale.shape[1]
    if x.shape[0] <= 16:
        most = (151.0 + (zero.abs().max().item() if zero is not None else 0)) * scale.double().repeat_interleave(group, 1)
        bound = ONE_ROUNDING * exact.abs() + 136 * 2.0 ** -24 * (x.double().abs() @ most.t())
        norm = ONE_ROUNDING
    else:
        spread = x.double().abs() @ w.abs().t()
        bound = ONE_ROUNDING * exact.abs() + (ONE_ROUNDING + (x.shape[1] + 16) * 2.0 ** -24) * spread
        norm = TWO_ROUNDINGS
    off = (y.double() - exact).abs()
    assert y.dtype == torch.bfloat16 and y.shape == exact.shape
    assert (off <= bound).all(), (off - bound).max()
    assert off.norm() <= norm * exact.norm(), off.norm() / exact.norm()


_SHAPES = [
    (1, 1, 32, 32), (1, 257, 64, 64), (2, 16, 128, 128), (16, 100, 4096, 128), (13, 1000, 2080, 32), (9, 4097, 11008, 64),
    (3, 70000, 256, 32), (16, 70000, 384, 128),              # rows: tiles of channels shared by a workgroup
    (17, 129, 288, 32), (33, 300, 1024, 128), (64, 128, 8192, 64), (65, 1000, 640, 128), (128, 257, 4160, 64),
    (200, 4096, 1024, 32), (129, 511, 160, 32), (300, 2048, 4096, 128), (777, 8200, 576, 64), (1030, 8190, 288, 32),
    (257, 30000, 1024, 128), (40, 28670, 4096, 64), (512, 8192, 2048, 128), (300, 1031, 64, 64),
]


@pytest.mark.parametrize("m,n,k,group", _SHAPES)
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_matches_float64(gpu, m, n, k, group, zeros):
    print(f"int4 linear: m={m} n={n} k={k} group={group} zeros={zeros}", flush=True)
    x, codes, scale, zero = _inputs(gpu, m, n, k, group, zeros)
    packed = hip.int4_pack(codes, scale, zero)
    _check(hip.int4_linear(x, *packed, n=n), x, codes, scale, zero)
    assert torch.equal(hip.int4_dequantize(*packed, n, k).double(), _weights(codes, scale, zero).float().double())


@pytest.mark.parametrize("m", [3, 40])
def test_strided_and_unaligned_rows(gpu, m):
    x, codes, scale, zero = _inputs(gpu, m, 200, 320, 64, True)
    packed = hip.int4_pack(codes, scale, zero)
    want = hip.int4_linear(x, *packed, n=200)
    for wide, offset in ((328, 8), (336, 0), (333, 0), (328, 3)):
        held = torch.full((m, wide), float("nan"), dtype=torch.bfloat16, device=gpu)
        rows = held[:, offset: offset + 320]
        rows.copy_(x)
        assert torch.equal(hip.int4_linear(rows, *packed, n=200), want)
    assert torch.equal(hip.int4_linear(x.t().contiguous().t(), *packed, n=200), want)
    one = x[:1].expand(m, 320)  # rows that are one
    assert torch.equal(hip.int4_linear(one, *packed, n=200), hip.int4_linear(one.contiguous(), *packed, n=200))


@pytest.mark.parametrize("m", [5, 50])
def test_rows_that_are_not_finite_stay_with_themselves(gpu, m):
    x, codes, scale, _ = _inputs(gpu, m, 100, 256, 32, False)
    packed = hip.int4_pack(codes, scale)
    want = hip.int4_linear(x, *packed, n=100)
    x[1, 3], x[3, 250] = float("nan"), float("inf")
    got = hip.int4_linear(x, *packed, n=100)
    others = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(got[others], want[others])
    assert got[1].isnan().all() and not got[3].isfinite().any()
    big = torch.full((m, 256), 1e30, dtype=torch.bfloat16, device=gpu)
    assert hip.int4_linear(big, *packed, n=100).isfinite().all()


def test_empty_calls_and_refusals(gpu):
    x, codes, scale, zero = _inputs(gpu, 4, 48, 128, 32, True)
    weight, s, z = hip.int4_pack(codes, scale, zero)
    assert hip.int4_linear(x[:0], weight, s, z).shape == (0, 48)
    assert hip.int4_linear(x, weight[:0], s[:0], z[:0]).shape == (4, 0)
    assert hip.int4_linear(x, weight, s, z).shape == (4, 48) and hip.int4_linear(x, weight, s, z, n=33).shape == (4, 33)
    for bad in (lambda: hip.int4_linear(x, weight, s, z, n=49), lambda: hip.int4_linear(x, weight, s, z, n=32),
                lambda: hip.int4_linear(x[:, :96], weight[:, :0], s, z), lambda: hip.int4_linear(x[0], weight, s, z),
                lambda: hip.int4_linear(x[:, :100], weight, s, z), lambda: hip.int4_linear(x, weight, s[..., :3], z),
                lambda: hip.int4_linear(x, weight, s, z[:1]), lambda: hip.int4_linear(x, weight[:, :, ::2], s, z),
                lambda: hip.int4_linear(x, weight.cpu(), s, z), lambda: hip.int4_linear(x[:, :0], weight[:, :0], s[:, :0]),
                lambda: hip.int4_linear(x.clone().requires_grad_(), weight, s, z),
                lambda: hip.int4_linear(x, weight, s.clone().requires_grad_(), z)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hip.int4_linear(x.half(), weight, s, z), lambda: hip.int4_linear(x, weight.to(torch.int32), s, z),
                lambda: hip.int4_linear(x, weight, s.float(), z)):
        with pytest.raises(TypeError):
            bad()
    with torch.no_grad():
        assert torch.equal(hip.int4_linear(x.requires_grad_(), weight, s, z), hip.int4_linear(x.detach(), weight, s, z))
