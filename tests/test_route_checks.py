"""Refusals of the routing operator (host checks, no GPU) and its oracle's own checks."""
import ctypes

import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc


def _desc(**kw):
    d = dict(rows=4, logits_ld=8, experts=8, top_k=2, score=0, groups=1, top_groups=1, renormalize=1,
             dtype=0, scale=1.0)
    d.update(kw)
    return _lib.CkanRouteDesc(*[d[n] for n, _ in _lib.CkanRouteDesc._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), _lib.CKAN_ERR_INVALID_ARG),
    (dict(experts=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(experts=513, logits_ld=513), _lib.CKAN_ERR_UNSUPPORTED),
    (dict(logits_ld=7), _lib.CKAN_ERR_INVALID_ARG),
    (dict(top_k=0), _lib.CKAN_ERR_INVALID_ARG),
    (dict(top_k=9), _lib.CKAN_ERR_INVALID_ARG),
    (dict(groups=3), _lib.CKAN_ERR_INVALID_ARG),
    (dict(groups=4, top_groups=5), _lib.CKAN_ERR_INVALID_ARG),
    (dict(groups=4, top_groups=1, top_k=3), _lib.CKAN_ERR_INVALID_ARG),
    (dict(score=2), _lib.CKAN_ERR_INVALID_ARG),
    (dict(dtype=7), _lib.CKAN_ERR_INVALID_ARG),
    (dict(scale=float("inf")), _lib.CKAN_ERR_INVALID_ARG),
])
def test_route_desc_refused(change, code):
    lib = _lib.load()
    d = _desc(**change)
    assert lib.ckan_route(ctypes.byref(d), 256, None, 256, 256, None) == code
    assert lib.ckan_last_error()
    assert lib.ckan_route_backward(ctypes.byref(d), 256, 256, 256, 256, None) == code


def test_route_null_pointers_and_empty():
    lib = _lib.load()
    assert lib.ckan_route(None, 256, None, 256, 256, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_route(_desc(), None, None, 256, 256, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_route(_desc(rows=0), None, None, None, None, None) == _lib.CKAN_OK


def test_route_python_refusals():
    with pytest.raises(ValueError, match="score"):
        kan_amd.functional.route(torch.zeros(2, 4), 1, score="relu")
    with pytest.raises(RuntimeError, match="rows, experts"):
        kan_amd.functional.route(torch.zeros(4), 1)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kan_amd.functional.route(torch.zeros(2, 4), 1)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_oracle_gradient_against_differences(score, renormalize):
    rng = np.random.RandomState(3)
    l = rng.randn(3, 7)
    _, idx = orc.route(l, 3, score)
    idx[1, 2] = -1
    dw = rng.randn(3, 3)
    got = orc.route_backward(l, idx, dw, score, renormalize, 1.7)

    def f(v):
        return (orc.route_weights(orc.route_scores(v, score)[0], idx, renormalize, 1.7) * dw).sum()

    h = 1e-6
    for at in np.ndindex(*l.shape):
        e = np.zeros_like(l)
        e[at] = h
        assert abs((f(l + e) - f(l - e)) / (2 * h) - got[at]) < 1e-8


def test_route_rows_within_a_launch():
    lib = _lib.load()
    d = _desc(rows=1 << 26)
    assert lib.ckan_route(d, 256, None, 256, 256, None) == _lib.CKAN_ERR_UNSUPPORTED
    assert lib.ckan_route_backward(d, 256, 256, 256, 256, None) == _lib.CKAN_ERR_UNSUPPORTED
