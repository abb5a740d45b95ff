"""The mixture layer inside torch's autocast: its gate, choice and weights stay fp32, as its own compute says."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("compute", ["fp32", "bf16"])
def test_autocast_changes_nothing(low, compute):
    torch.manual_seed(0)
    layer = kan_amd.MixtureKANLayer(40, 30, 4, experts=8, top_k=2, compute=compute).cuda()
    x = torch.randn(100, 40, device="cuda")
    want = layer(x)
    want_grads = torch.autograd.grad(want.square().sum(), list(layer.parameters()))
    with torch.autocast("cuda", dtype=low):
        got = layer(x)
    # outside, as torch asks: inside, it would cast the products of its own backward too
    grads = torch.autograd.grad(got.square().sum(), list(layer.parameters()))
    assert got.dtype == torch.float32 and torch.equal(got, want)
    for a, b in zip(grads, want_grads):
        assert torch.equal(a, b)
