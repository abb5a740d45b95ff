"""Gradients of rows whose upstream gradients differ by many powers of two, each row held to its own size.

The bounds are those of test_gpu_experts.py, on each row's error over the row's norm: fp32 5e-6, bf16 5e-3.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 5e-6, torch.bfloat16: 5e-3}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,in_dim,out,degree,experts,top_k", [(150, 40, 33, 5, 2, 1), (90, 64, 130, 8, 3, 2), (70, 9, 20, 11, 1, 1)])
def test_rows_of_small_gradients(rows, in_dim, out, degree, experts, top_k, dtype):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, in_dim, generator=g).to(dtype)
    c = (torch.randn(experts, in_dim, out, degree + 1, generator=g) / in_dim).to(dtype)
    idx = torch.rand(rows, experts, generator=g).topk(top_k, 1)[1]
    w = torch.rand(rows, top_k, generator=g).add(0.5)
    dy = (torch.randn(rows, out, generator=g) * 2.0 ** -(torch.arange(rows) % 8 * 9).view(-1, 1)).to(dtype)  # to 2^-63
    xd, cd, wd = (v.cuda().requires_grad_() for v in (x, c, w))
    y = kan_amd.functional.kan_experts(xd, cd, idx.cuda(), wd)
    dx, dc, dw = (v.double().cpu().numpy() for v in torch.autograd.grad(y, (xd, cd, wd), dy.cuda()))
    _, rx, rc, rw = orc.kan_experts(*(v.double().numpy() for v in (x, c)), idx.numpy(), w.double().numpy(), dy.double().numpy())
    tol = TOL[dtype]
    assert (np.linalg.norm(dx - rx, axis=1) <= tol * np.linalg.norm(rx, axis=1)).all()
    # a weight's gradient is one dot product: its terms' rounding counts against the norms of its factors
    z = np.abs(rw).max()
    size = np.linalg.norm(dy.double().numpy(), axis=1) * np.sqrt(out) * max(1.0, z)
    assert (np.abs(dw - rw).max(1) <= tol * size).all()
    assert np.linalg.norm(dc - rc) <= tol * np.linalg.norm(rc)
