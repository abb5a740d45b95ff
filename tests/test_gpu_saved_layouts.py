"""Every saved tensor, parameters, statistics, targets and indices among them, comes back from its hook strided: the gradients
are those of a pass without hooks."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).requires_grad_()


def residual(dim=50, rows=20, gate_rows=False):
    x, y = randn(rows, dim, seed=1), randn(rows, dim, seed=2)
    gate = randn(rows, dim, seed=3) if gate_rows else randn(dim, seed=3)
    vectors = [randn(dim, seed=s) for s in range(4, 8)]
    out, h = f.residual_norm(x, y, norm="layer", gate=gate, post_weight=vectors[0], post_bias=vectors[1],
                             next_weight=vectors[2], next_bias=vectors[3], dropout=0.2, dropout_state=3)
    return out.square().sum() + h.sin().sum(), (x, y, gate, *vectors)


def residual_gate_rows():
    return residual(gate_rows=True)


def residual_wide():
    return residual(9000, 4)


def log_probs():
    l = randn(20, 70, seed=8)
    got = f.log_probs(l, torch.arange(20, device="cuda"))
    return (got.logp * got.entropy).sum(), (l,)


def experts():
    x, coeffs, weights = randn(30, 24, seed=9), randn(5, 24, 16, 4, seed=10), randn(30, 2, seed=11)
    indices = torch.randint(0, 5, (30, 2), device="cuda", generator=torch.Generator("cuda").manual_seed(12))
    return f.kan_experts(x, coeffs, indices, weights).sin().sum(), (x, coeffs, weights)


def route():
    l = randn(20, 16, seed=13)
    return f.route(l, 4)[0].square().sum(), (l,)


@pytest.mark.parametrize("call", [residual, residual_gate_rows, residual_wide, log_probs, experts, route], ids=lambda c: c.__name__)
def test_saved_tensors_that_come_back_strided(call):
    loss, leaves = call()
    want = torch.autograd.grad(loss, leaves)
    seen = []

    def strided(t):
        seen.append(t.shape)
        return torch.stack([t, torch.zeros_like(t)], -1)[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), strided):
        loss, leaves = call()
    got = torch.autograd.grad(loss, leaves)
    assert seen
    for a, b in zip(got, want):
        assert torch.equal(a, b)
