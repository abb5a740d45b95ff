"""Orthogonalisation of coefficients as they lie, [in, out, D] taken as the matrix [out, in D], through the C-ABI.

Bounds: fp32 1e-5 (test_gpu_ortho.py derives it); bf16 adds its rounding, at most 2^-8 of a value.
"""
import numpy as np
import pytest
import torch

from kan_amd import _lib
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 1e-5 + 2.0 ** -8}
CODE = {torch.float32: _lib.CKAN_DTYPE_F32, torch.bfloat16: _lib.CKAN_DTYPE_BF16}


def _call(x, batch, rows, cols, inner, strides, steps=5):
    lib = _lib.load()
    desc = _lib.CkanOrthoDesc(*strides, batch, rows, cols, inner, steps, CODE[x.dtype], 3.4445, -4.7750, 2.0315, 1e-7)
    need = lib.ckan_orthogonalize_workspace_bytes(desc)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.full_like(x, float("nan"))
    _lib.check(lib.ckan_orthogonalize(desc, x.data_ptr(), out.data_ptr(), ws.data_ptr(), need, _lib.stream_ptr(x.device)))
    return out


# out < in D (wide), out > in D (tall), a side of at most 64, several matrices
@pytest.mark.parametrize("experts,in_dim,out,d", [(1, 40, 70, 5), (1, 64, 130, 9), (1, 20, 150, 4), (2, 33, 200, 3),
                                                  (1, 300, 80, 9), (2, 9, 20, 5), (1, 9, 40, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_coefficients_as_they_lie(experts, in_dim, out, d, dtype):
    g = torch.Generator().manual_seed(in_dim + out)
    c = torch.randn(experts, in_dim, out, d, generator=g).to(dtype)
    got = _call(c.cuda(), experts, out, in_dim * d, d, (in_dim * out * d, d, out * d, 1)).double().cpu().numpy()
    for e in range(experts):
        want = orc.orthogonalize(orc.coeff_matrix(c[e].double().numpy()))
        assert np.linalg.norm(orc.coeff_matrix(got[e]) - want) <= TOL[dtype] * np.linalg.norm(want)
