"""The mixture layer: routing, experts and Muon together, against the 64-bit oracle."""
import os
import sys

import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("score,groups,top_groups", [("softmax", 1, 1), ("sigmoid", 4, 2)])
def test_layer_against_definition(score, groups, top_groups):
    torch.manual_seed(2)
    layer = kan_amd.MixtureKANLayer(20, 12, 5, experts=8, top_k=3, score=score, groups=groups, top_groups=top_groups)
    x = torch.randn(90, 20)
    logits = (x @ layer.gate.detach().t()).double().numpy()
    w, idx = orc.route(logits, 3, score=score, groups=groups, top_groups=top_groups)
    want = orc.kan_experts(x.numpy(), layer.cheby_coeffs.detach().numpy(), idx, w)
    y = layer.cuda()(x.cuda()).detach().double().cpu().numpy()
    # the experts' 5e-6 and the gate's product in fp32 (20 terms), whose error passes to the weights
    assert np.linalg.norm(y - want) <= 1e-5 * np.linalg.norm(want)


def test_bf16_layer_and_gradients_flow():
    torch.manual_seed(3)
    layer = kan_amd.MixtureKANLayer(64, 48, 8, experts=4, top_k=2, compute="bf16").cuda()
    x = torch.randn(300, 64, device="cuda", requires_grad=True)
    y = layer(x)
    assert y.dtype == torch.float32
    y.square().mean().backward()
    for g in (x.grad, layer.gate.grad, layer.cheby_coeffs.grad):
        assert torch.isfinite(g).all() and g.abs().sum() > 0
    layer.compute = "fp32"
    z = layer(x)
    assert ((y - z).norm() / z.norm()).item() <= 2e-2  # the framework's bf16 bound


def test_balance_moves_towards_unused_experts():
    torch.manual_seed(4)
    layer = kan_amd.MixtureKANLayer(6, 5, 3, experts=4, top_k=1, score="sigmoid", balance=True).cuda()
    with torch.no_grad():
        layer.gate[2] = 0.0  # sigmoid 0.5 for every row
    layer(torch.randn(400, 6, device="cuda"))
    load = torch.bincount(layer._last_indices.reshape(-1), minlength=4).float()
    layer.update_balance(0.01)
    assert torch.equal(layer.balance_bias, 0.01 * torch.sign(load.mean() - load))
    assert "balance_bias" in layer.state_dict()


def test_example_trains_and_serves():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_mixture
    finally:
        sys.path.pop(0)
    model, losses = train_mixture.train(steps=60, rows=2048, log=None)
    assert np.mean(losses[-5:]) < 0.6 * np.mean(losses[:5])
    # single rows take the streaming form, the batch the same sums in another order
    assert train_mixture.serve(model).abs().max().item() <= 1e-4
