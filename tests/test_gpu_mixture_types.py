"""kan_mixture's two forms on rows and coefficients of different types: one accuracy on either side of the rule between
them, and with gradients.

y against the 64-bit sum for the call's own weights and choice: 5e-6 of its norm, the bound of either form's fp32 results
(coefficients in bf16 are exact in fp32), and half a step more of each value of a y in bf16. Gradients: those of the same
call on the coefficients widened before it, that of the coefficients rounded to their type.
"""
import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
F32, BF16 = torch.float32, torch.bfloat16


def make(rows, x_dtype, c_dtype, experts=4, in_dim=60, out_dim=46, degree=5):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, in_dim, generator=g).to(x_dtype)
    gate = 2 * torch.randn(experts, in_dim, generator=g) / in_dim ** 0.5
    coeffs = (torch.randn(experts, in_dim, out_dim, degree + 1, generator=g) / (in_dim * (degree + 1))).to(c_dtype)
    return x.cuda(), gate.cuda(), coeffs.cuda()


@pytest.mark.parametrize("x_dtype,c_dtype", [(F32, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("rows,few,grad", [(63, 1, False), (64, 0, False), (64, 0, True), (1, 1, False), (1, 1, True), (500, 0, False)])
def test_both_forms_keep_the_rows_accuracy(x_dtype, c_dtype, rows, few, grad):
    x, gate, coeffs = make(rows, x_dtype, c_dtype)
    desc = _lib.CkanMixtureDesc(rows, 4, 4, 60, 46, 5, 0, 1, 1, 1, 0, 0, 0, 1.0)
    assert _lib.load().ckan_mixture_few(desc) == few
    y, w, idx = f.kan_mixture(x.requires_grad_(grad), gate, coeffs, 4)
    assert y.dtype == x_dtype and y.requires_grad == grad
    want = orc.kan_experts(x.detach().double().cpu().numpy(), coeffs.double().cpu().numpy(), idx.cpu().numpy(),
                           w.detach().double().cpu().numpy())
    err = np.abs(y.detach().double().cpu().numpy() - want)
    if x_dtype == BF16:
        err = np.maximum(err - 2.0 ** -8 * np.abs(want), 0)
    assert np.linalg.norm(err) <= 5e-6 * np.linalg.norm(want)


def test_gradients_of_mixed_types():
    x, gate, coeffs = make(37, F32, BF16)
    up = torch.randn(37, 46, device="cuda")

    def grads(c):
        leaves = [t.detach().requires_grad_() for t in (x, gate, c)]
        y, _, _ = f.kan_mixture(*leaves, 2)
        return y, *torch.autograd.grad(y, leaves, up)

    y, dx, dgate, dc = grads(coeffs)
    z, ex, egate, ec = grads(coeffs.float())
    assert torch.equal(y, z) and torch.equal(dx, ex) and torch.equal(dgate, egate)
    assert dc.dtype == BF16 and torch.equal(dc, ec.bfloat16())
