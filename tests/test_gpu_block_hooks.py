"""Saved tensors that come back in another layout: inputs with a row pitch of their own, kept on the host between the
passes, return dense, and the gradients are those of a pass without hooks."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def sliced(rows, dim, seed, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(rows, 3 * dim, device="cuda", generator=g).to(dtype)[:, dim + 1:2 * dim + 1].requires_grad_()


def residual():
    x, y, gate = (sliced(20, 50, s) for s in range(3))
    w = torch.ones(50, device="cuda", requires_grad=True)
    out, h = f.residual_norm(x, y, post_weight=w, gate=gate, next_weight=w, dropout=0.2, dropout_state=3)
    return out.square().sum() + h.sin().sum(), (x, y, gate, w)


def wide():
    x, w = sliced(5, 9000, 4), torch.ones(9000, device="cuda", requires_grad=True)
    return f.row_norm(x, w).sin().sum(), (x, w)


def log_probs():
    l = sliced(20, 70, 5, torch.bfloat16)
    got = f.log_probs(l, torch.arange(20, device="cuda"))
    return (got.logp * got.entropy).sum(), (l,)


def dropout():
    x = sliced(20, 70, 6)
    return f.dropout(x, 0.4, 8).square().sum(), (x,)


def route():
    l = sliced(20, 16, 7)
    w, _ = f.route(l, 4)
    return w.square().sum(), (l,)


@pytest.mark.parametrize("call", [residual, wide, log_probs, dropout, route], ids=lambda c: c.__name__)
def test_saved_on_the_host(call):
    loss, leaves = call()
    want = torch.autograd.grad(loss, leaves)
    with torch.autograd.graph.save_on_cpu():
        loss, leaves = call()
    for a, b in zip(torch.autograd.grad(loss, leaves), want):
        assert torch.equal(a, b)
