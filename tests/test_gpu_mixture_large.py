"""Tensors past 2^31 elements: what lies beyond gives the same as the same values in small tensors."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional

# bf16 results of the same sums in another order: a rounding here and there (half an ulp, 2^-8, of few values)
TOL = 2.0 ** -8


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_coefficients_past_32_bits():
    experts, dim, degree = 60, 2048, 8
    c = torch.randn(experts, dim, dim, degree + 1, device="cuda", dtype=torch.bfloat16).div_(dim)
    assert c.numel() > 2 ** 31
    last = c[58:].clone()
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(20, dim, device="cuda", generator=g).bfloat16()
    idx, w = torch.tensor([[59, 58]] * 20, device="cuda"), torch.rand(20, 2, device="cuda", generator=g)
    with torch.no_grad():  # the coefficients read as they lie
        assert _rel(f.kan_experts(x, c, idx, w), f.kan_experts(x, last, idx - 58, w)) <= TOL
    x = torch.randn(600, dim, device="cuda", generator=g).bfloat16()  # packed, and their gradient
    idx, w = torch.randint(58, 60, (600, 1), device="cuda", generator=g), torch.ones(600, 1, device="cuda")
    dy = torch.randn(600, dim, device="cuda", generator=g).bfloat16()
    grads = []
    for coeffs, first in ((c, 0), (last, 58)):
        leaf, cl = x.clone().requires_grad_(), coeffs.requires_grad_()
        y = f.kan_experts(leaf, cl, idx - first, w)
        gx, gc = torch.autograd.grad(y, (leaf, cl), dy)
        grads.append((y.detach(), gx, gc[58 - first:]))
        if not first:
            assert (gc[:58] == 0).all()
    for a, b in zip(*grads):
        assert _rel(a, b) <= TOL


def test_logits_past_32_bits():
    l = torch.randn(4300000, 512, device="cuda", dtype=torch.bfloat16)
    assert l.numel() > 2 ** 31
    tail = l[-500:].clone().requires_grad_()
    l.requires_grad_()
    w, idx = f.route(l, 4)
    wt, it = f.route(tail, 4)
    assert torch.equal(w[-500:], wt) and torch.equal(idx[-500:], it)
    dw = torch.randn(l.shape[0], 4, device="cuda")
    g, = torch.autograd.grad(w, l, dw)
    gt, = torch.autograd.grad(wt, tail, dw[-500:])
    assert torch.equal(g[-500:], gt)


def test_matrices_past_32_bits():
    x = torch.randn(3, 64, 1 << 24, device="cuda", dtype=torch.bfloat16)
    got = f.orthogonalize(x)
    assert torch.equal(got[2], f.orthogonalize(x[2].clone()))
