"""Biases that are not finite: they move the choice, never a score."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_bias_without_a_value(score, groups, top_groups):
    g = torch.Generator().manual_seed(groups)
    logits = torch.randn(50, 16, generator=g)
    bias = torch.zeros(16)
    bias[3], bias[9], bias[6] = float("nan"), -float("inf"), float("inf")
    l = logits.cuda().requires_grad_()
    w, idx = kan_amd.functional.route(l, 3, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups)
    s = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    idx = idx.cpu()
    assert not ((idx == 3) | (idx == 9)).any() and (idx[:, 0] == 6).all()
    # the weights are the chosen experts' scores over their sum; a softmax's sum holds every expert's
    chosen = s.gather(1, idx)
    assert (w.detach().double().cpu() - chosen / chosen.sum(1, keepdim=True)).abs().max() <= 1e-6
    raw, again = kan_amd.functional.route(l, 3, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups, renormalize=False)
    assert torch.equal(again.cpu(), idx) and (raw.detach().double().cpu() - chosen).abs().max() <= 1e-6
    dw = torch.randn(50, 3, generator=g)
    dl, = torch.autograd.grad(raw, l, dw.cuda())
    leaf = logits.double().requires_grad_()
    t = torch.softmax(leaf, 1) if score == "softmax" else torch.sigmoid(leaf)
    want, = torch.autograd.grad(t.gather(1, idx), leaf, dw.double())
    assert (dl.double().cpu() - want).abs().max() <= 4e-6 * want.abs().max()
