"""Refusals of the residual-block, dropout and log-probability operators (host checks, no GPU), and their oracle's own checks."""
import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwad

import kan_amd
from kan_amd import _lib
from oracle import block_oracle as orc

f = kan_amd.functional
INVALID, UNSUPPORTED = _lib.CKAN_ERR_INVALID_ARG, _lib.CKAN_ERR_UNSUPPORTED


def _struct(cls, base, change):
    d = {**base, **change}
    return cls(**d)


RESIDUAL = dict(rows=4, x_ld=8, y_ld=8, gate_ld=8, dim=8, eps=1e-6, scale=1.0)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), INVALID), (dict(rows=1 << 32), UNSUPPORTED), (dict(dim=0), INVALID),
    (dict(dim=(1 << 20) + 1), UNSUPPORTED), (dict(x_dtype=2), INVALID), (dict(y_dtype=-1), INVALID),
    (dict(gate_dtype=9), INVALID), (dict(next_bias_dtype=3), INVALID), (dict(norm=2), INVALID),
    (dict(gate_rows=2), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(dropout=1.5), INVALID), (dict(dropout=float("nan")), INVALID),
    (dict(x_ld=-8), INVALID), (dict(gate_ld=-1), INVALID),
])
def test_residual_desc_refused(change, code):
    lib = _lib.load()
    d = _struct(_lib.CkanResidualDesc, RESIDUAL, change)
    b = _lib.CkanResidualBuffers(x=256, y=256, next_weight=256, out=256, h=256, stats=256, dout=256, dx=256)
    assert lib.ckan_residual_forward(d, b, None) == code
    assert lib.ckan_last_error()
    assert lib.ckan_residual_backward(d, b, 256, 1 << 30, None) == code
    if "dropout" not in change:
        assert lib.ckan_residual_stats_bytes(d) == 0 and lib.ckan_residual_workspace_bytes(d) == 0


@pytest.mark.parametrize("buffers", [
    dict(), dict(x=256), dict(x=256, y=256), dict(x=256, next_weight=256), dict(x=256, next_weight=256, h=256, gate=256),
    dict(x=256, next_weight=256, h=256, post_weight=256), dict(x=256, y=256, out=256, post_bias=256),
    dict(x=256, y=256, out=256, next_bias=256), dict(x=256, y=256, out=256, h=256), dict(x=256, next_weight=256, h=256, out=256),
    dict(x=257, y=256, out=256), dict(x=256, y=258, out=256), dict(x=256, y=256, out=256, gate=255),
    dict(x=256, y=256, out=256, stats=8), dict(x=256, y=256, out=256, dropout_state=4),
])
def test_residual_forward_buffers_refused(buffers):
    lib = _lib.load()
    d = _lib.CkanResidualDesc(**RESIDUAL)
    assert lib.ckan_residual_forward(d, _lib.CkanResidualBuffers(**buffers), None) == INVALID


@pytest.mark.parametrize("buffers", [
    dict(), dict(dh=256), dict(dy=256, y=None), dict(dgate=256), dict(dpost_weight=256), dict(dpost_bias=256),
    dict(dnext_weight=256), dict(dnext_bias=256), dict(dx=257), dict(dx=256, dout_ld=-1), dict(dx=256, dh_ld=-8),
])
def test_residual_backward_buffers_refused(buffers):
    lib = _lib.load()
    d = _lib.CkanResidualDesc(**RESIDUAL)
    base = dict(x=256, y=256, dout=256)
    if buffers:
        base["stats"] = 256
    assert lib.ckan_residual_backward(d, _lib.CkanResidualBuffers(**{**base, **buffers}), 256, 1 << 30, None) == INVALID


def test_residual_workspace_and_empty():
    lib = _lib.load()
    d = _lib.CkanResidualDesc(**RESIDUAL)
    b = _lib.CkanResidualBuffers(x=256, y=256, dout=256, stats=256, dx=256)
    need = lib.ckan_residual_workspace_bytes(d)
    assert need > 0 and lib.ckan_residual_stats_bytes(d) == 4 * 16 + 16
    assert lib.ckan_residual_backward(d, b, 256, need - 1, None) == _lib.CKAN_ERR_WORKSPACE
    assert lib.ckan_residual_backward(d, b, None, need, None) == INVALID
    assert lib.ckan_residual_backward(d, b, 264, need, None) == INVALID
    assert lib.ckan_residual_forward(None, b, None) == INVALID and lib.ckan_residual_forward(d, None, None) == INVALID
    d.rows = 0
    assert lib.ckan_residual_forward(d, _lib.CkanResidualBuffers(), None) == _lib.CKAN_OK
    assert lib.ckan_residual_backward(d, b, None, 0, None) == _lib.CKAN_OK
    b.dnext_weight = 256  # nothing is written, zeros are the caller's
    assert lib.ckan_residual_backward(d, b, None, 0, None) == INVALID


DROPOUT = dict(rows=4, dim=8, x_ld=8, p=0.5)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), INVALID), (dict(dim=0), INVALID), (dict(x_ld=-1), INVALID), (dict(p=-0.1), INVALID),
    (dict(p=1.1), INVALID), (dict(p=float("nan")), INVALID), (dict(dtype=2), INVALID),
    (dict(rows=1 << 32), UNSUPPORTED), (dict(dim=(1 << 34) + 1), UNSUPPORTED),
])
def test_dropout_desc_refused(change, code):
    assert _lib.load().ckan_dropout(_struct(_lib.CkanDropoutDesc, DROPOUT, change), None, 256, 256, None, None) == code


def test_dropout_pointers_refused():
    lib, d = _lib.load(), _lib.CkanDropoutDesc(**DROPOUT)
    for args in ((None, None, 256, None), (None, 256, None, None), (None, 258, 256, None), (4, 256, 256, None),
                 (None, 256, 256, 4)):
        assert lib.ckan_dropout(d, *args, None) == INVALID
    assert lib.ckan_dropout(None, None, 256, 256, None, None) == INVALID
    d.rows = 0
    assert lib.ckan_dropout(d, None, None, None, None, None) == _lib.CKAN_OK


LOGP = dict(rows=4, logits_ld=8, classes=8, top=2)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), INVALID), (dict(classes=0), INVALID), (dict(top=-1), INVALID), (dict(top=9), INVALID),
    (dict(top=65, classes=100), UNSUPPORTED), (dict(dtype=2), INVALID), (dict(logits_ld=-1), INVALID),
    (dict(rows=1 << 31), UNSUPPORTED), (dict(classes=(1 << 30) + 1), UNSUPPORTED),
])
def test_log_probs_desc_refused(change, code):
    lib, d = _lib.load(), _struct(_lib.CkanLogProbsDesc, LOGP, change)
    assert lib.ckan_log_probs(d, 256, 256, 256, 256, 256, 256, None, 256, 1 << 30, None) == code
    assert lib.ckan_log_probs_backward(d, 256, 256, 256, 256, 256, 256, None) == code
    assert lib.ckan_log_probs_workspace_bytes(d) == 0


def test_log_probs_pointers_refused():
    lib, d = _lib.load(), _lib.CkanLogProbsDesc(**LOGP)
    ok = [256] * 6
    for i in range(6):
        bad = ok[:i] + [None] + ok[i + 1:]
        assert lib.ckan_log_probs(d, *bad, None, 256, 1 << 30, None) == INVALID
    assert lib.ckan_log_probs(d, 257, *ok[1:], None, 256, 1 << 30, None) == INVALID
    for i in (0, 1, 2, 5):
        args = [256] * 6
        args[i] = None
        assert lib.ckan_log_probs_backward(d, *args, None) == INVALID
    d.rows = 0
    assert lib.ckan_log_probs(d, *[None] * 7, None, 0, None) == _lib.CKAN_OK
    assert lib.ckan_log_probs_backward(d, *[None] * 6, None) == _lib.CKAN_OK


X, W = torch.zeros(2, 4), torch.ones(4)


@pytest.mark.parametrize("call,error,match", [
    (lambda: f.row_norm(X, W), RuntimeError, "ROCm device"),
    (lambda: f.row_norm(X, W, norm="batch"), ValueError, "norm"),
    (lambda: f.row_norm(torch.tensor(1.0), W), RuntimeError, "dim >= 1"),
    (lambda: f.row_norm(torch.zeros(2, 0), torch.ones(0)), RuntimeError, "dim >= 1"),
    (lambda: f.residual_norm(X, X), RuntimeError, "ROCm device"),
    (lambda: f.dropout(X, 0.5, 1), RuntimeError, "ROCm device"),
    (lambda: f.dropout(torch.tensor(1.0), 0.5, 1), RuntimeError, "scalar"),
    (lambda: f.log_probs(X, torch.zeros(2, dtype=torch.int64)), RuntimeError, "ROCm device"),
    (lambda: f.log_probs(X, torch.zeros(3, dtype=torch.int64)), RuntimeError, "targets must be"),
    (lambda: f.log_probs(X, torch.zeros(2)), RuntimeError, "int64"),
    (lambda: f.log_probs(torch.zeros(2, 0), torch.zeros(2, dtype=torch.int64)), RuntimeError, "classes"),
])
def test_python_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_sizes_past_the_descriptors_32_bits_are_refused():
    meta = dict(device="meta")
    with pytest.raises(RuntimeError, match="2\\^20"):
        f.row_norm(torch.zeros(1, 2 ** 32 + 8, **meta), W)
    for classes, top in ((2 ** 32 + 8, 0), (100, 2 ** 32 + 1), (100, -1)):
        with pytest.raises(RuntimeError, match="2\\^30 classes"):
            f.log_probs(torch.zeros(1, classes, **meta), torch.zeros(1, dtype=torch.int64, **meta), top=top)


@pytest.mark.parametrize("call", [
    lambda d: f.row_norm(d, W), lambda d: f.residual_norm(X, d), lambda d: f.residual_norm(d, X),
    lambda d: f.dropout(d, 0.5, 1), lambda d: f.log_probs(d, torch.zeros(2, dtype=torch.int64)),
])
def test_tangents_are_refused(call):
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fwad.make_dual(X, torch.ones_like(X)))


# ---- the oracle -----------------------------------------------------------------------

def test_philox_known_answers():
    """The published known-answer vectors of Philox 4x32-10 (counter and key of zeros, of ones), through the words
    that the mask is made of."""
    def words(counter, key):
        c, k = list(counter), list(key)
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c

    assert words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    # element (row 3, column 13) of call 5 under seed 2^32 + 9: chunk 1, half 5 of its words
    hi, lo = words([1, 3, 5, 0], [9, 1]), words([1, 3, 5, 1 << 31], [9, 1])
    number = (hi[2] >> 16) << 16 | lo[2] >> 16
    for p, kept in ((number / 2 ** 32, True), ((number + 1) / 2 ** 32, False)):
        assert orc.keep_mask(2 ** 32 + 9, 5, 4, 20, p)[3, 13] == kept


def test_mask_frequencies():
    # 2^17 elements: a count's standard deviation is sqrt(n p (1 - p)); five of them
    for p in (0.0, 0.001, 0.25, 0.9, 1.0):
        kept = orc.keep_mask(77, 3, 64, 2048, p)
        n = kept.size
        assert abs(kept.sum() - n * (1 - p)) <= 5 * np.sqrt(n * p * (1 - p))


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("gate_rows", [False, True])
def test_residual_oracle_against_differences(norm, gate_rows):
    rng = np.random.RandomState(4)
    rows, dim, p = 3, 6, 0.25
    v = {"x": rng.randn(rows, dim), "y": rng.randn(rows, dim), "gate": rng.randn(*((rows, dim) if gate_rows else (dim,)))}
    v.update({k: rng.randn(dim) for k in ("post_weight", "post_bias", "next_weight", "next_bias")})
    keep = orc.keep_mask(1, 0, rows, dim, p)
    dout, dh = rng.randn(rows, dim), rng.randn(rows, dim)
    kw = dict(norm=norm, eps=1e-3, scale=0.7, keep=keep, p=p)
    got = orc.residual(**v, **kw, dout=dout, dh=dh)

    def loss(w):
        r = orc.residual(**w, **kw)
        return (r["out"][0] * dout).sum() + (r["h"][0] * dh).sum()

    for name, t in v.items():
        for at in np.ndindex(*t.shape):
            step = np.zeros_like(t)
            step[at] = 1e-6
            diff = (loss({**v, name: t + step}) - loss({**v, name: t - step})) / 2e-6
            assert abs(diff - got[name][0][at]) < 1e-6, name


def test_log_probs_oracle_against_differences():
    rng = np.random.RandomState(5)
    l = 2 * rng.randn(4, 6)
    l[1, 2] = -np.inf
    t = np.array([2, 0, -100, 5])
    dl, dH = rng.randn(4), rng.randn(4)
    got, size = orc.log_probs_backward(l, t, dl, dH)
    assert (np.abs(got) <= size + 1e-15).all()

    def loss(v):
        logp, h, *_ = orc.log_probs(v, t)
        return (logp * dl).sum() + (h * dH).sum()

    for at in np.ndindex(*l.shape):
        if l[at] == -np.inf:
            assert got[at] == 0
            continue
        step = np.zeros_like(l)
        step[at] = 1e-6
        assert abs((loss(l + step) - loss(l - step)) / 2e-6 - got[at]) < 1e-8


# ---- the mixture layer for few rows -----------------------------------------------------

MIXTURE = dict(rows=2, experts=4, top_k=2, in_dim=8, out_dim=6, degree=3, groups=1, top_groups=1, renormalize=1, scale=1.0)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), INVALID), (dict(experts=0), INVALID), (dict(experts=513), UNSUPPORTED), (dict(top_k=0), INVALID),
    (dict(top_k=5), INVALID), (dict(in_dim=0), INVALID), (dict(out_dim=0), INVALID), (dict(degree=0), UNSUPPORTED),
    (dict(degree=17), UNSUPPORTED), (dict(score=2), INVALID), (dict(groups=3), INVALID), (dict(top_groups=2), INVALID),
    (dict(x_dtype=2), INVALID), (dict(gate_dtype=2), INVALID), (dict(coeff_dtype=2), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(rows=2000), UNSUPPORTED), (dict(rows=64, experts=2), UNSUPPORTED),
])
def test_mixture_desc_refused(change, code):
    lib, d = _lib.load(), _struct(_lib.CkanMixtureDesc, MIXTURE, change)
    assert lib.ckan_mixture_few(d) == 0 and lib.ckan_mixture_workspace_bytes(d) == 0
    assert lib.ckan_mixture_forward(d, 256, 256, 256, None, 256, 256, 256, 256, 1 << 30, None) == code


def test_mixture_pointers_refused():
    lib, d = _lib.load(), _lib.CkanMixtureDesc(**MIXTURE)
    need = lib.ckan_mixture_workspace_bytes(d)
    assert lib.ckan_mixture_few(d) == 1 and need > 0
    for i in (0, 1, 2, 4, 5, 6, 7):
        args = [256, 256, 256, None, 256, 256, 256, 256]
        args[i] = None
        assert lib.ckan_mixture_forward(d, *args, need, None) == INVALID
    for i in (0, 1, 2, 4, 7):
        args = [256, 256, 256, None, 256, 256, 256, 256]
        args[i] = 264
        assert lib.ckan_mixture_forward(d, *args, need, None) == INVALID
    args = [256, 256, 256, None, 256, 256, 256, 256]
    assert lib.ckan_mixture_forward(d, *args, need - 1, None) == _lib.CKAN_ERR_WORKSPACE
    d.rows = 0
    assert lib.ckan_mixture_few(d) == 0
    assert lib.ckan_mixture_forward(d, *[None] * 8, 0, None) == _lib.CKAN_OK


def test_mixture_python_refusals():
    x, gate, coeffs = torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(3, 4, 5, 2)
    with pytest.raises(ValueError, match="score"):
        f.kan_mixture(x, gate, coeffs, 1, score="relu")
    with pytest.raises(RuntimeError, match="ROCm device"):
        f.kan_mixture(x, gate, coeffs, 1)
    with fwad.dual_level():
        for i in range(3):
            args = [x, gate, coeffs]
            args[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f.kan_mixture(*args, 1)
