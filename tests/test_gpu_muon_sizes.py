"""Muon's step on matrices with both sides above 64, in every layout that it takes, against the 64-bit oracle.

Bound: five steps in fp32 1e-5 of the update's norm (test_gpu_ortho.py derives it), the update being lr of a matrix; the
parameters here are of the update's size, so that its error shows.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

TOL = 1e-5
LR = 0.02


def _inputs(shape, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randn(*shape, generator=g) * 1e-3
    grad = torch.randn(*shape, generator=g) * 1e-3
    buf = torch.randn(*shape, generator=g) * 1e-3
    return p, grad, buf


def _check(shape, p, g, buf, pd, bd, **kw):
    for e in range(shape[0]) if len(shape) == 4 else [slice(None)]:
        want_p, want_b = orc.muon_step(p[e].numpy(), g[e].numpy(), buf[e].numpy(), **kw)
        got_p, got_b = pd[e].double().cpu().numpy(), bd[e].double().cpu().numpy()
        update = np.linalg.norm(want_p - p[e].double().numpy())
        assert np.linalg.norm(got_p - want_p) <= TOL * update + 2.0 ** -23 * np.linalg.norm(want_p)
        assert np.linalg.norm(got_b - want_b) <= 1e-6 * np.linalg.norm(want_b)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [
    (130, 200), (200, 130), (96, 96),     # ordinary matrices, wide, tall and square
    (513, 66), (66, 2500),                # odd rows (no vector store), two steps a pass
    (40, 70, 5), (64, 100, 9), (70, 77, 3),  # coefficients: out < in D, gathered
    (20, 150, 4), (30, 301, 3),           # out > in D
    (300, 80, 9),                         # two steps a pass
    (3, 48, 96, 9), (2, 25, 130, 4),      # experts, wide and tall
    (70, 90, 1),                          # degree 0
])
def test_step(shape, nesterov):
    p, g, buf = _inputs(shape, sum(shape))
    pd, bd = p.cuda(), buf.cuda()
    kan_amd.optim.muon_step_(pd, g.cuda(), bd, lr=LR, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    _check(shape, p, g, buf, pd, bd, lr=LR, momentum=0.9, nesterov=nesterov, weight_decay=0.1)


@pytest.mark.parametrize("shape", [(130, 200), (64, 100, 9), (2, 25, 130, 4)])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_addresses_that_no_vector_load_takes(shape, which):
    p, g, buf = _inputs(shape, which)
    on_device = []
    for k, t in enumerate((p, g, buf)):
        store = torch.zeros(t.numel() + 4, device="cuda")
        off = 1 if k == which else 0
        view = store[off:off + t.numel()].view(shape)
        view.copy_(t)
        on_device.append((store, view, off))
    kan_amd.optim.muon_step_(on_device[0][1], on_device[1][1], on_device[2][1], lr=LR, momentum=0.9)
    _check(shape, p, g, buf, on_device[0][1], on_device[2][1], lr=LR, momentum=0.9)
    for store, view, off in on_device:  # nothing beside the tensors is written
        assert (store[off + view.numel():] == 0).all() and (off == 0 or store[0] == 0)


@pytest.mark.parametrize("shape", [(64, 48), (20, 33, 5), (130, 200), (64, 100, 9)])
@pytest.mark.parametrize("steps", [0, 1, 7, 12])
def test_other_step_counts(shape, steps):
    p, g, buf = _inputs(shape, steps)
    pd, bd = p.cuda(), buf.cuda()
    kan_amd.optim.muon_step_(pd, g.cuda(), bd, lr=LR, momentum=0.9, steps=steps)
    # the iteration's own amplification from five steps to twelve is below 20 for full-rank matrices
    want_p, _ = orc.muon_step(p.numpy(), g.numpy(), buf.numpy(), LR, 0.9, True, 0.0, steps=steps)
    update = np.linalg.norm(want_p - p.double().numpy())
    assert np.linalg.norm(pd.double().cpu().numpy() - want_p) <= 20 * TOL * update + 2.0 ** -23 * np.linalg.norm(want_p)


def test_optimizer_of_a_wide_layer():
    """Five optimizer steps of a layer whose matrix has both sides above 64, against the oracle's."""
    torch.manual_seed(3)
    layer = kan_amd.ChebyKANLayer(40, 72, 4).cuda()
    opt = kan_amd.optim.Muon(layer.parameters(), lr=LR, weight_decay=0.01)
    p = layer.cheby_coeffs.detach().cpu().double().numpy()
    buf = np.zeros_like(p)
    for k in range(5):
        x = torch.randn(128, 40, device="cuda")
        opt.zero_grad()
        layer(x).square().mean().backward()
        g = layer.cheby_coeffs.grad.cpu().numpy()
        opt.step()
        p, buf = orc.muon_step(p, g, buf, LR, 0.95, True, 0.01)
    got = layer.cheby_coeffs.detach().cpu().double().numpy()
    assert np.linalg.norm(got - p) <= 5 * TOL * np.linalg.norm(p)
