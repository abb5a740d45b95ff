"""Gradients of renormalised weights whose upstream gradients share an offset: it has no part in the result.

Bound as in test_gpu_route.py: 4e-6 of the row's largest entry (exactly representable dw, so that the 64-bit reference
sees the same differences).
"""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu


def _reference(logits, idx, dw, score):
    leaf = logits.double().requires_grad_()
    s = torch.softmax(leaf, 1) if score == "softmax" else torch.sigmoid(leaf)
    c = s.gather(1, idx)
    g, = torch.autograd.grad(c / (c.sum(1, keepdim=True) + 1e-20), leaf, dw.double())
    return g


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(20, 1), (8, 2), (130, 6)])
def test_a_shared_offset_cancels(experts, top_k, score):
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn(300, experts, generator=g)
    dw = torch.round(torch.randn(300, top_k, generator=g) * 64) / 64 + 2.0 ** 12
    l = logits.cuda().requires_grad_()
    w, idx = kan_amd.functional.route(l, top_k, score=score)
    got, = torch.autograd.grad(w, l, dw.cuda())
    got = got.double().cpu()
    if top_k == 1:  # the one weight is 1 whatever the logits
        assert (got == 0).all()
        return
    # of the differences: with the offset, 64 bits leave 2^12 2^-53 where they are all zero;
    # its own part, offset 1e-20 / sum^2, is below the last term
    want = _reference(logits, idx.cpu(), dw - dw[:, :1], score)
    assert ((got - want).abs().max(1).values <= 4e-6 * want.abs().max(1).values + 2.0 ** 12 * 1e-20 / 0.01).all()


def test_equal_gradients_give_none():
    g = torch.Generator().manual_seed(1)
    l = torch.randn(64, 33, generator=g).cuda().requires_grad_()
    w, _ = kan_amd.functional.route(l, 5)
    got, = torch.autograd.grad(w, l, torch.full((64, 5), 0.3, device="cuda"))
    assert (got == 0).all()


def test_rows_whose_scores_underflow():
    """Scores near and below the 1e-20 that their sum is divided with: a slot alone has a gradient then."""
    logits = torch.tensor([[-44.0, -90.0], [-46.5, -90.0], [-50.0, -90.0], [-33.0, -90.0]])
    for top_k in (1, 2):
        l = logits.cuda().requires_grad_()
        w, idx = kan_amd.functional.route(l, top_k, score="sigmoid")
        dw = torch.full((4, top_k), 0.7)
        got, = torch.autograd.grad(w, l, dw.cuda())
        want = _reference(logits, idx.cpu(), dw, "sigmoid")
        assert ((got.double().cpu() - want).abs().max(1).values <= 4e-6 * want.abs().max(1).values).all()
