"""The mixture layer's forward is its parts', bit for bit, wherever the few-row form does not take it, on parameters of either type."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def layer_of(compute, dtype):
    torch.manual_seed(3)
    layer = kan_amd.MixtureKANLayer(40, 30, 5, experts=8, top_k=2, score="sigmoid", balance=True, compute=compute).cuda()
    layer.balance_bias += 0.1 * torch.arange(8, device="cuda").remainder(3)
    layer.cheby_coeffs.data = layer.cheby_coeffs.data.to(dtype)
    return layer


@pytest.mark.parametrize("compute", ["fp32", "bf16"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,grad", [(3, True), (700, True), (700, False), (0, False)])
def test_the_layer_is_its_parts(compute, dtype, rows, grad):
    layer = layer_of(compute, dtype)
    x, up = torch.randn(rows, 40, device="cuda"), torch.randn(rows, 30, device="cuda")
    with torch.set_grad_enabled(grad):
        y = layer(x)
        weights, indices = f.route(x @ layer.gate.t(), 2, score="sigmoid", bias=layer.balance_bias)
        at = torch.float32 if compute == "fp32" else torch.bfloat16
        z = f.kan_experts(x.to(at), layer.cheby_coeffs.to(at), indices, weights).to(torch.float32)
    assert y.dtype == torch.float32 and torch.equal(y, z) and torch.equal(layer._last_indices, indices)
    if grad:
        for a, b in zip(torch.autograd.grad(y, layer.parameters(), up), torch.autograd.grad(z, layer.parameters(), up)):
            assert torch.equal(a, b)
    layer.update_balance()


@pytest.mark.parametrize("compute", ["fp32", "bf16"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_few_rows(compute, dtype, rows):
    layer = layer_of(compute, dtype)
    x = torch.randn(rows, 40, device="cuda")
    with torch.no_grad():
        want = f.kan_mixture(x, layer.gate, layer.cheby_coeffs, 2, score="sigmoid", bias=layer.balance_bias)
        assert torch.equal(layer(x), want[0]) and torch.equal(layer._last_indices, want[2])


def test_a_frozen_layer_gives_gradients_of_its_input():
    layer = layer_of("fp32", torch.float32).requires_grad_(False)
    x = torch.randn(5, 40, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(layer(x).sum(), x)
    assert torch.isfinite(g).all() and g.abs().sum() > 0
    assert not layer(x.detach()).requires_grad
