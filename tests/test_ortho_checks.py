"""Refusals of the orthogonalisation and Muon's step (host checks, no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc


def _desc(**kw):
    d = dict(batch_stride=32, row_stride=8, outer_stride=1, inner_stride=0, batch=1, rows=4, cols=8, inner=1,
             steps=5, dtype=0, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7)
    d.update(kw)
    return _lib.CkanOrthoDesc(*[d[n] for n, _ in _lib.CkanOrthoDesc._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), _lib.CKAN_ERR_INVALID_ARG),
    (dict(batch=65536), _lib.CKAN_ERR_INVALID_ARG),
    (dict(rows=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(cols=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(rows=16385, cols=16385), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(inner=3), _lib.CKAN_ERR_INVALID_ARG),
    (dict(inner=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(row_stride=-8), _lib.CKAN_ERR_INVALID_ARG),
    (dict(steps=-1), _lib.CKAN_ERR_INVALID_ARG),
    (dict(steps=101), _lib.CKAN_ERR_INVALID_ARG),
    (dict(dtype=2), _lib.CKAN_ERR_INVALID_ARG),
    (dict(eps=-1.0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(a=float("nan")), _lib.CKAN_ERR_INVALID_ARG),
    (dict(a=4.0, b=1.0, c=1.0), _lib.CKAN_ERR_UNSUPPORTED),   # singular values grow without bound
])
def test_desc_refused(change, code):
    lib = _lib.load()
    d = _desc(**change)
    assert lib.ckan_orthogonalize(ctypes.byref(d), 256, 256, 256, 1 << 30, None) == code
    assert lib.ckan_last_error()
    assert lib.ckan_muon_step(ctypes.byref(d), 256, 256, 256, 0.1, 0.9, 0.0, 1.0, 1, 256, 1 << 30, None) == code
    assert lib.ckan_orthogonalize_workspace_bytes(ctypes.byref(d)) == 0


def test_workspace_and_pointers():
    lib = _lib.load()
    d = _desc()
    need = lib.ckan_orthogonalize_workspace_bytes(d)
    assert need > 0
    assert lib.ckan_orthogonalize(d, 256, 256, 256, need - 1, None) == _lib.CKAN_ERR_WORKSPACE
    assert lib.ckan_orthogonalize(d, None, 256, 256, need, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_orthogonalize(d, 256, 256, None, need, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_orthogonalize(d, 256, 256, 264, need, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_orthogonalize(_desc(batch=0), None, None, None, 0, None) == _lib.CKAN_OK
    assert lib.ckan_muon_step(d, 256, None, 256, 0.1, 0.9, 0.0, 1.0, 1, 256, need, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_muon_step(d, 256, 256, 256, 0.1, 1.0, 0.0, 1.0, 1, 256, need, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_muon_step(_desc(dtype=1), 256, 256, 256, 0.1, 0.9, 0.0, 1.0, 1, 256, need,
                              None) == _lib.CKAN_ERR_INVALID_ARG


def test_python_refusals():
    with pytest.raises(RuntimeError, match="rows, cols"):
        kan_amd.functional.orthogonalize(torch.zeros(4))
    with pytest.raises(RuntimeError, match="ROCm device"):
        kan_amd.functional.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="matrices"):
        kan_amd.optim.Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="momentum"):
        kan_amd.optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], momentum=1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kan_amd.optim.muon_step_(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4), lr=0.1)


def test_oracle_iterates_the_singular_values():
    rng = np.random.RandomState(0)
    g = rng.randn(9, 23)
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / (np.linalg.norm(s) + 1e-7)
    for _ in range(5):
        s = s * (3.4445 - 4.7750 * s ** 2 + 2.0315 * s ** 4)
    assert np.abs(orc.orthogonalize(g) - (u * s) @ vt).max() < 1e-12
    assert np.abs(orc.orthogonalize(g.T).T - orc.orthogonalize(g)).max() < 1e-12
