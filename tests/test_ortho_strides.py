"""Strides by which the matrices of a batch would share elements are refused (host check, no GPU)."""
import ctypes

import pytest

from kan_amd import _lib


def _desc(batch, stride):
    return _lib.CkanOrthoDesc(stride, 8, 1, 0, batch, 4, 8, 1, 5, 0, 3.4445, -4.7750, 2.0315, 1e-7)


@pytest.mark.parametrize("stride", [0, 1, 31])
def test_overlapping_matrices_are_refused(stride):
    lib = _lib.load()
    d = _desc(2, stride)
    assert lib.ckan_orthogonalize(ctypes.byref(d), 256, 256, 256, 1 << 30, None) == _lib.CKAN_ERR_INVALID_ARG
    assert b"batch_stride" in lib.ckan_last_error()
    assert lib.ckan_muon_step(ctypes.byref(d), 256, 256, 256, 0.1, 0.9, 0.0, 1.0, 1, 256, 1 << 30, None) == _lib.CKAN_ERR_INVALID_ARG
    assert lib.ckan_orthogonalize_workspace_bytes(ctypes.byref(d)) == 0


@pytest.mark.parametrize("batch,stride", [(1, 0), (2, 32), (3, 40)])
def test_others_are_taken(batch, stride):
    assert _lib.load().ckan_orthogonalize_workspace_bytes(_desc(batch, stride)) > 0
