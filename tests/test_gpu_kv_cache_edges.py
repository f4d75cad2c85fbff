"""The 8-bit cache and the int8 linear at the edges of their contracts: scales of zero, infinities, the largest
numbers, gradients that are asked for, memory that runs out. Against float64, and on the types of errors."""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import workloads as W

pytestmark = pytest.mark.gpu


def test_a_layer_whose_scales_were_rounded_runs_in_torch(gpu):
    """``module.bfloat16()`` rounds the channel scales, which the kernels take in fp32."""
    lin = W.init_normal_(W.Int8Linear(64, 32), seed=1).to(gpu).bfloat16()
    x = torch.randn(5, 64, device=gpu, generator=torch.Generator(device=gpu).manual_seed(0)).bfloat16()
    want = lin.cpu()(x.cpu())
    lin = lin.to(gpu)
    assert (lin(x).cpu().float() - want.float()).norm() <= 2.0 ** -8 * want.float().norm()
    assert W.int8_group(x, [lin, lin]) is None
