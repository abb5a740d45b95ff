"""Refusals of the experts' products (host checks, no GPU) and the oracle's own checks."""
import ctypes

import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import chebykan_oracle
from oracle import mixture_oracle as orc


def _desc(**kw):
    d = dict(rows=4, experts=3, top_k=2, in_dim=5, out_dim=6, degree=4, dtype=0, wdtype=0)
    d.update(kw)
    return _lib.CkanExpertsDesc(*[d[n] for n, _ in _lib.CkanExpertsDesc._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), _lib.CKAN_ERR_INVALID_ARG),
    (dict(rows=1 << 29), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(experts=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(experts=513), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(top_k=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(top_k=65), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(in_dim=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(out_dim=65537), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(degree=-1), _lib.CKAN_ERR_INVALID_ARG),
    (dict(degree=0), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(degree=17), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(dtype=2), _lib.CKAN_ERR_INVALID_ARG),
    (dict(wdtype=-1), _lib.CKAN_ERR_INVALID_ARG),
])
def test_desc_refused(change, code):
    lib = _lib.load()
    d = _desc(**change)
    big = 1 << 40
    assert lib.ckan_experts_forward(ctypes.byref(d), 256, 256, 256, 256, 256, None, 256, big, None) == code
    assert lib.ckan_last_error()
    assert lib.ckan_experts_backward(ctypes.byref(d), 256, 256, 256, 256, 256, 256, 256, 256, big, None) == code
    assert lib.ckan_experts_saved_bytes(ctypes.byref(d)) == 0
    assert lib.ckan_experts_workspace_bytes(ctypes.byref(d), 0, 1) == 0


def test_workspace_and_pointers():
    lib = _lib.load()
    d = _desc()
    need, need_b = lib.ckan_experts_workspace_bytes(d, 0, 0), lib.ckan_experts_workspace_bytes(d, 1, 0)
    alone = lib.ckan_experts_workspace_bytes(d, 0, 1)
    assert alone > 0 and need > 0 and need_b > 0 and lib.ckan_experts_saved_bytes(d) > 0
    inv, ws = _lib.CKAN_ERR_INVALID_ARG, _lib.CKAN_ERR_WORKSPACE
    assert lib.ckan_experts_forward(d, 256, 256, 256, 256, 256, 256, 256, need - 1, None) == ws
    assert lib.ckan_experts_forward(d, 256, 256, 256, 256, 256, None, 256, alone - 1, None) == ws
    assert lib.ckan_experts_forward(d, None, 256, 256, 256, 256, None, 256, alone, None) == inv
    assert lib.ckan_experts_forward(d, 256, 256, 256, 256, 256, 264, 256, need, None) == inv
    assert lib.ckan_experts_forward(d, 256, 256, 256, 256, 256, None, None, alone, None) == inv
    assert lib.ckan_experts_forward(d, 256, 260, 256, 256, 256, None, 256, alone, None) == inv
    assert lib.ckan_experts_backward(d, 256, 256, 256, 256, 256, 256, 256, 256, need_b - 1, None) == ws
    assert lib.ckan_experts_backward(d, 256, 256, 256, 258, 256, 256, 256, 256, need_b, None) == inv
    assert lib.ckan_experts_backward(d, 256, 256, None, 256, 256, 256, 256, 256, need_b, None) == inv
    assert lib.ckan_experts_backward(d, 256, 256, 256, 256, None, None, None, None, 0, None) == _lib.CKAN_OK
    z = _desc(rows=0)
    assert lib.ckan_experts_forward(z, None, None, None, None, None, None, None, 0, None) == _lib.CKAN_OK
    assert lib.ckan_experts_backward(z, None, None, None, None, None, None, None, None, 0, None) == _lib.CKAN_OK
    assert lib.ckan_experts_backward(z, None, None, None, None, None, 256, None, None, 0, None) == inv


def test_python_refusals():
    f = kan_amd.functional.kan_experts
    x, c = torch.zeros(3, 4), torch.zeros(2, 4, 5, 3)
    i, w = torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 1)
    with pytest.raises(RuntimeError, match="ROCm device"):
        f(x, c, i, w)


def test_oracle_is_the_layer_for_one_expert():
    rng = np.random.RandomState(2)
    x, c = rng.randn(7, 5), rng.randn(1, 5, 6, 9)
    dy = rng.randn(7, 6)
    y, dx, dc, dw = orc.kan_experts(x, c, np.zeros((7, 1), dtype=np.int64), np.ones((7, 1)), dy)
    ry, rdx, rdc = chebykan_oracle.layer_forward_backward(*(torch.tensor(v) for v in (x, c[0], dy)))
    for a, b in ((y, ry), (dx, rdx), (dc[0], rdc)):
        assert np.abs(a - b.numpy()).max() < 1e-10
    assert np.abs(dw[:, 0] - (y * dy).sum(1)).max() < 1e-12


def test_oracle_gradients_against_differences():
    rng = np.random.RandomState(4)
    x, c, w, dy = rng.randn(4, 3), rng.randn(3, 3, 2, 5), rng.rand(4, 2), rng.randn(4, 2)
    idx = np.array([[0, 1], [2, 2], [-1, 0], [1, 5]])
    grads = orc.kan_experts(x, c, idx, w, dy)[1:]
    args = [x, c, w]
    for k in range(3):
        u = rng.randn(*args[k].shape)

        def f(s):
            v = list(args)
            v[k] = v[k] + s * 1e-6 * u
            return (orc.kan_experts(v[0], v[1], idx, v[2]) * dy).sum()

        assert abs((f(1) - f(-1)) / 2e-6 - (grads[k] * u).sum()) < 1e-7


@pytest.mark.parametrize("change", [dict(rows=1 << 26, top_k=2), dict(rows=1 << 24, top_k=1, in_dim=513),
                                    dict(rows=1 << 24, top_k=1, out_dim=513)])
def test_sizes_within_a_launch(change):
    lib = _lib.load()
    assert lib.ckan_experts_workspace_bytes(_desc(**change), 0, 1) == 0
    assert b"above 2^" in lib.ckan_last_error()
