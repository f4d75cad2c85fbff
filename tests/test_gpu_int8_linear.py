"""The int8 linear: codes and integer sums bit for bit, outputs against float64.

The sums are exact, so an output differs from the exact product of codes and scales by three roundings: two fp32
multiplications and the conversions (2^-24 each) and one to bf16 (2^-9 of the value at most, half a unit in the last
of 8 bits): ``ONE_ROUNDING`` bounds each element.
"""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import hip

pytestmark = pytest.mark.gpu

ONE_ROUNDING = 2.0 ** -8


def _inputs(gpu, m, n, k, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + m + 3 * n + 7 * k)
    x = torch.randn(m, k, device=gpu, generator=g)
    x[:, :: max(1, k // 8)] *= 8.0
    w = torch.randn(n, k, device=gpu, generator=g).mul(32).round().clamp(-127, 127).to(torch.int8)
    scale = torch.exp(0.2 * torch.randn(n, device=gpu, generator=g)) * 1e-3
    return x.bfloat16(), w, scale


def _quantised(x):
    """The definition in 32 bits, on the CPU."""
    x = x.cpu().float()
    top = x.abs().amax(-1, keepdim=True)
    made = top * torch.tensor(1 / 127, dtype=torch.float32)
    scale = torch.where(made < 2.0 ** -100, 0.0, made)
    codes = (x * torch.where(scale > 0, 1.0 / scale, 0.0)).round().clamp(-127, 127)
    bad = ~top.isfinite()
    return codes.masked_fill(bad, 0).nan_to_num(0).to(torch.int8), scale.masked_fill(bad, float("nan"))[:, 0]


@pytest.mark.parametrize("m,k", [(1, 16), (3, 256), (5, 272), (17, 4096), (2, 131072), (1, 11008)])
def test_quantize_is_the_definition(gpu, m, k):
    x = _inputs(gpu, m, 1, k)[0]
    x[-1, k // 2] = 300.0
    codes, scales = hip.int8_quantize(x)
    want, want_scales = _quantised(x)
    assert torch.equal(codes[:, :k].cpu(), want) and not codes[:, k:].any()
    assert torch.equal(scales.cpu(), want_scales)


def test_quantize_of_extreme_rows(gpu):
    """Zeros, numbers below the smallest scale, the largest number, ties, an infinity, a NaN; rows of a wider
    tensor."""
    wide = torch.zeros(7, 96, device=gpu, dtype=torch.bfloat16)
    x = wide[:, 16:80]
    x[1] = 1e-32
    x[2, ::2], x[2, 1] = torch.finfo(torch.bfloat16).max, -torch.finfo(torch.bfloat16).max
    x[3] = torch.arange(64) - 0.5
    x[3, 0] = 127.0
    x[4, 3], x[5, 7], x[6, 1] = float("inf"), float("nan"), float("-inf")
    codes, scales = hip.int8_quantize(x)
    want, want_scales = _quantised(x)
    assert torch.equal(codes[:, :64].cpu(), want)
    assert torch.equal(scales.cpu().nan_to_num(9.0), want_scales.nan_to_num(9.0))
    w = torch.ones(40, 64, dtype=torch.int8, device=gpu)
    y = hip.int8_linear(x, w, torch.ones(40, device=gpu))
    assert y[4:].isnan().all() and not y[:2].any() and y[3].isfinite().all()
    assert y[2].isinf().all()  # 31 times the largest number


_SHAPES = [
    (1, 1, 16), (1, 257, 272), (2, 16, 256), (16, 100, 4096), (13, 1000, 2064), (9, 4096, 11008),   # up to 16 rows
    (17, 129, 272), (33, 300, 1040), (64, 128, 8192), (65, 1000, 640), (128, 257, 4112), (200, 4096, 1024),
    (129, 511, 144), (300, 2048, 4096), (777, 8200, 528), (2111, 8190, 272), (257, 30000, 1040),  # tiles of 64 tokens
    (13, 28672, 8192), (200, 28670, 4096), (100, 28672, 8192),                  # of 64 and 128, K split or not
    (300, 30001, 1040), (512, 8192, 28672),                                     # of 256
]


@pytest.mark.parametrize("m,n,k", _SHAPES)
def test_linear_matches_exact_sums(gpu, m, n, k):
    x, w, scale = _inputs(gpu, m, n, k)
    codes, want_scales = _quantised(x)
    got = hip.int8_linear(x, w, scale).cpu().double()
    want = codes.to(gpu).double() @ w.double().t() * want_scales[:, None].to(gpu).double() * scale.double()
    want = want.cpu()
    assert ((got - want).abs() <= ONE_ROUNDING * want.abs()).all()


@pytest.mark.parametrize("m,n,k", [
    (1, 30000, 4112), (1, 300, 32768), (2, 20000, 8208), (4, 17, 272), (7, 9001, 272), (8, 8200, 4096),  # rounds x itself
    (16, 40, 2048), (16, 9001, 3600), (3, 20000, 8208), (12, 9001, 8208), (1, 5000, 131072),              # codes from a launch
])
def test_rows_of_a_wider_tensor_as_codes_and_product(gpu, m, n, k):
    """However the codes come to the product: the same numbers, of rows among others, one of them zeros, one with an
    infinity."""
    x, w, scale = _inputs(gpu, m, n, k)
    wide = torch.full((m, k + 64), 3.0e38, device=gpu, dtype=torch.bfloat16)
    wide[:, :k] = x
    if m > 2:
        wide[1, :k] = 0.0
        wide[2, k - 1] = float("-inf")
    codes, scales = _quantised(wide[:, :k])
    want = codes.to(gpu).double() @ w.double().t() * scales[:, None].to(gpu).double() * scale.double()
    got = hip.int8_linear(wide[:, :k], w, scale)
    assert torch.equal(got.view(torch.int16), hip.int8_matmul(*hip.int8_quantize(wide[:, :k]), w, scale).view(torch.int16))
    rest = [i for i in range(m) if m <= 2 or i != 2]
    assert ((got.double() - want).abs() <= ONE_ROUNDING * want.abs())[rest].all()
    if m > 2:
        assert got[2].isnan().all()


@pytest.mark.parametrize("m,n,k", [(0, 5, 16), (3, 0, 16), (3, 5, 0), (20, 130, 0), (1, 1, 0)])
def test_linear_of_nothing(gpu, m, n, k):
    x = torch.ones(m, k, device=gpu, dtype=torch.bfloat16)
    w = torch.ones(n, k, device=gpu, dtype=torch.int8)
    scale = torch.ones(n, device=gpu)
    for got in (hip.int8_linear(x, w, scale), hip.int8_matmul(*hip.int8_quantize(x), w, scale)):
        assert got.shape == (m, n) and not got.any()


def test_linear_of_the_largest_sums(gpu):
    """Every product 127^2: the longest K reaches 2113929216 of the 2147483647 that 32 bits hold."""
    k = hip.INT8_LINEAR_MAX_K
    for m in (2, 40):
        x = torch.ones(m, k, device=gpu, dtype=torch.bfloat16)
        x[1] = -1.0
        w = torch.full((3, k), 127, dtype=torch.int8, device=gpu)
        w[1] = -127
        got = hip.int8_linear(x, w, torch.ones(3, device=gpu)).cpu().double()
        want = x.cpu()[:, :1].double() * 127.0 * k * torch.tensor([1.0, -1.0, 1.0], dtype=torch.float64)
        assert ((got - want).abs() <= ONE_ROUNDING * want.abs()).all()


def test_shared_input_is_quantised_once(gpu):
    """int8_matmul of one quantised input gives the bits of int8_linear for each weight, on another stream too."""
    x, w, scale = _inputs(gpu, 40, 512, 1024)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        codes, scales = hip.int8_quantize(x)
        got = [hip.int8_matmul(codes, scales, part, s) for part, s in ((w[:256], scale[:256]), (w[256:], scale[256:]))]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(torch.cat(got, 1), hip.int8_linear(x, w, scale))
