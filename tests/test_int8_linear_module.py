"""The int8 projection as a module, on the host: what its inputs' gradients are, and which calls the kernels take."""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import workloads as W


def _layer(k=64, n=32):
    return W.init_normal_(W.Int8Linear(k, n), seed=1)


def _weight64(lin):
    return lin.weight.double() * lin.scale.detach().double()[:, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_input_gets_the_gradient_of_the_product(dtype):
    """g @ (W * scale): within the rounding of its type (2^-8 of a bf16 number; 2^-24 of each of 32 products and
    their sums in fp32). The outputs are those of a call without a gradient."""
    torch.manual_seed(0)
    lin = _layer()
    x = torch.randn(3, 5, 64).to(dtype)
    want = lin(x)
    x.requires_grad_()
    y = lin(x)
    assert torch.equal(y, want)
    g = torch.randn_like(y)
    y.backward(g)
    exact = g.double() @ _weight64(lin)
    bound = 2.0 ** -8 * exact.abs() + 64 * 2.0 ** -24 * (g.double().abs() @ _weight64(lin).abs())
    assert x.grad.dtype == dtype and ((x.grad.double() - exact).abs() <= bound).all()


def test_the_gradient_is_the_slope_across_the_steps_of_the_rounding():
    """A difference over many steps: each of its two ends is off by half a step s / 2 of x at most."""
    torch.manual_seed(1)
    lin = _layer()
    x = torch.randn(4, 64)
    x[:, 0] = 8.0  # the row's scale, whatever the others do
    x.requires_grad_()
    lin(x).sum().backward()
    w = _weight64(lin).sum(0)
    h, step = 1.0, 8.0 / 127
    for j in (1, 17, 63):
        shift = torch.zeros(64)
        shift[j] = h
        with torch.no_grad():
            slope = (lin(x + shift) - lin(x - shift)).double().sum(-1) / (2 * h)
        bound = step / (2 * h) * _weight64(lin).abs().sum(0)[j] + 1e-5
        assert ((slope - x.grad[:, j].double()).abs() <= bound).all()
        assert ((x.grad[:, j].double() - w[j]).abs() <= 1e-5).all()


def test_transforms_see_the_same_derivative():
    torch.manual_seed(2)
    lin = _layer()
    x, one = torch.randn(3, 5, 64), torch.ones(3, 5, 64)
    w = _weight64(lin).float()
    assert torch.allclose(torch.func.jvp(lin, (x,), (one,))[1], one @ w.t(), atol=1e-5)
    grads = torch.vmap(torch.func.grad(lambda a: lin(a).sum()))(x)
    assert torch.allclose(grads, torch.ones(3, 5, 32) @ w, atol=1e-5)


def test_a_trained_scale_keeps_its_gradient():
    torch.manual_seed(3)
    lin = _layer()
    lin.scale.requires_grad_()
    x = torch.randn(6, 64)
    (want,) = torch.autograd.grad(lin(x).sum(), lin.scale)  # the product over the scale
    x.requires_grad_()
    lin(x).sum().backward()
    assert torch.equal(lin.scale.grad, want)
    assert torch.allclose(want, lin(x.detach()).detach().sum(0) / lin.scale.detach(), rtol=1e-4)


def test_a_decoder_of_int8_projections_passes_gradients_on():
    """Through a layer's seven projections: near the gradient of the weights that their codes stand for. Each
    projection rounds its input (steps of about 3 / 127 sigma, an error of 0.7% of sigma), which moves the gradients
    of what follows by little; a tenth is far from that and from a gradient that is lost."""
    shape = W.LlamaShape(n_layers=1, hidden=64, n_heads=2, n_kv_heads=1, head_dim=32, inter=96, int8=True)
    layer = W.init_normal_(W.DecoderLayer(shape, torch.float32), seed=4, std=0.1)
    plain = W.DecoderLayer(W.LlamaShape(**{**shape.__dict__, "int8": False}), torch.float32)
    with torch.no_grad():
        for norm in (layer.attn_norm, layer.mlp_norm, plain.attn_norm, plain.mlp_norm):
            norm.weight.fill_(1.0)
        for name, mod in layer.named_modules():
            if isinstance(mod, W.Int8Linear):
                plain.get_submodule(name).weight.copy_(mod.weight.float() * mod.scale[:, None])
    torch.manual_seed(4)
    data, g = torch.randn(1, 8, 64), torch.randn(1, 8, 64)
    grads = []
    for mod in (layer, plain):
        x = data.clone().requires_grad_()
        mod(x, 0, torch.ones(8, 32), torch.zeros(8, 32), torch.zeros(1, 8, 1, 32), torch.zeros(1, 8, 1, 32)).backward(g)
        grads.append(x.grad - g)  # less the residual's own
    assert (grads[0] - grads[1]).norm() <= 0.1 * grads[1].norm()


def test_a_scale_of_another_type_is_not_for_the_kernel(monkeypatch):
    lin = _layer()
    monkeypatch.setattr(W.hip, "kernel_call", lambda *tensors: True)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    assert lin.kernel_eligible(x)
    assert not lin.bfloat16().kernel_eligible(x)
