"""What the 4-bit linear of up to 32 rows leaves of weights that are 0, under inputs of which a few are large.

The kernel sums x (128 + c) and takes (128 + z) sum x off: products are exact, and each of the up to 128 + 8 additions of
a group and behind it loses up to 2^-24 of numbers up to 143 + 128 + |z| times the scale and sum |x|. That is no share of
the weights' own terms: weights of 0 leave it too.
"""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,zeros", [(128, False), (128, True), (64, False), (64, True), (32, False), (32, True)])
@pytest.mark.parametrize("m,n,k", [(1, 300, 512), (4, 4096, 1024), (16, 9000, 256), (25, 4096, 512), (32, 300, 2048)])
def test_weights_of_0_leave_no_more_than_the_sums_rounding(gpu, m, n, k, group, zeros):
    print(f"int4 zero weights: m={m} n={n} k={k} group={group} zeros={zeros}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(m + n + k)
    x = torch.randn(m, k, device=gpu, generator=g)
    x[:, :: k // 4] *= 3000.0
    x = x.bfloat16()
    codes = torch.randint(0, 16, (n, k), device=gpu, generator=g)
    zero = torch.randint(0, 16, (n, k // group), device=gpu, generator=g) if zeros else torch.full((n, k // group), 8, device=gpu)
    of_input = zero.repeat_interleave(group, 1)
    codes[::2] = of_input[::2]                                 # channels of nothing but 0
    large = torch.zeros(k, dtype=torch.bool, device=gpu)
    large[:: k // 4] = True
    codes = torch.where(large, of_input, codes)                # and 0 under the large inputs of the others
    scale = (torch.rand(n, k // group, device=gpu, generator=g) * 0.02 + 0.001).bfloat16()
    weight = (codes - of_input).double() * scale.double().repeat_interleave(group, 1)
    want = x.double() @ weight.T
    got = hip.int4_linear(x, *hip.int4_pack(codes, scale, zero.bfloat16() if zeros else None), n=n).double()
    most = (271.0 + zero.double()) * scale.double()
    bound = 136 * 2.0 ** -24 * (x.double().abs().unflatten(1, (-1, group)).sum(-1) @ most.T)
    off = (got - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + bound).all(), (off - bound).max()
    assert not want[:, ::2].any()
