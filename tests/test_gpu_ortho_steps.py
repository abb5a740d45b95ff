"""Newton-Schulz iterations of many steps, and of matrices without full rank, against the definition in 64 bits.

The bound follows each singular value s through the iteration, s -> s p(s^2), p(y) = a + b y + c y^2.  A step is the
difference of a X and (b A + c A^2) X, either up to a |X|, of operands that carry 2^-22 and sums of as much: it adds an
error whose Frobenius norm is at most 2^-20 a of the iterate's, spread over the m directions of the shorter side (two
steps in one pass: a^2, what the first step's error is after the second).  The next step multiplies what is
there by at most the larger of |d/ds s p(s^2)| (along the direction) and |p(s^2)| (across it).  The bound is the norm
of the sum over the result's.
Directions of equal rows are no part of it: nothing may tell equal rows apart.  The definition is evaluated on the
singular values: by products, 64 bits leave an error of 2^-53 3.4^steps in the directions of singular values of zero
(0.06 of the result at 30 steps).  bf16 results add their own
rounding, at most 2^-8 of a value, and 2^-9 for steps taken as a product of m x m matrices (the limit that the
kernels' rule sets).
"""
import numpy as np
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)


def _bound(g, steps, eps=1e-7, coefficients=NS):
    a, b, c = coefficients
    s = np.linalg.svd(g, compute_uv=False)
    s = s[s > 1e-13 * s[0]] / (np.linalg.norm(s) + eps)
    d, m = np.zeros_like(s), min(g.shape)
    for _ in range(steps):
        step = 2.0 ** -20 * a * np.linalg.norm(s) / np.sqrt(m)
        y = s * s
        p = a + b * y + c * y * y
        d = d * np.maximum(np.abs(p + 2 * y * (b + 2 * c * y)), np.abs(p)) + step
        s = s * p
    return np.linalg.norm(d) / np.linalg.norm(s)


def _definition(g, steps, eps=1e-7, coefficients=NS):
    a, b, c = coefficients
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = np.where(s > 1e-13 * s[0], s, 0.0) / (np.linalg.norm(s) + eps)
    for _ in range(steps):
        y = s * s
        s = s * (a + b * y + c * y * y)
    return (u * s) @ vt


def _matrix(kind, rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    full = torch.randn(rows, cols, generator=g)
    if kind == "full":
        return full
    if kind == "low rank":
        return full[:, :rows // 8] @ torch.randn(rows // 8, cols, generator=g)
    if kind == "rank one":
        return full[:, :1] @ torch.randn(1, cols, generator=g)
    if kind == "equal halves":  # equal rows lie in different tiles
        return full[torch.arange(rows) % ((rows + 1) // 2)]
    if kind == "equal pairs":
        return full[torch.arange(rows) // 2]
    if kind == "four decades":
        u, _, v = torch.linalg.svd(full.double(), full_matrices=False)
        return ((u * 10.0 ** torch.linspace(0, -4, u.shape[1], dtype=torch.float64)) @ v).float()
    raise KeyError(kind)


def _check(got, g, steps, extra=0.0, **kw):
    want = _definition(g.double().numpy(), steps, **kw)
    v = got.double().cpu().numpy()
    assert np.isfinite(v).all()
    assert np.linalg.norm(v - want) <= (_bound(g.double().numpy(), steps, **kw) + extra) * np.linalg.norm(want)


def _equal_rows(got, kind, rows):
    first = torch.arange(rows) % ((rows + 1) // 2) if kind == "equal halves" else torch.arange(rows) // 2 * 2
    assert torch.equal(got, got[first.cuda()])


@pytest.mark.parametrize("steps", [12, 20, 30])
@pytest.mark.parametrize("kind", ["equal halves", "equal pairs"])
@pytest.mark.parametrize("rows,cols", [(200, 1500), (150, 151), (400, 900)])
def test_equal_rows_stay_equal(rows, cols, kind, steps):
    g = _matrix(kind, rows, cols, rows + steps)
    got = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    _equal_rows(got, kind, rows)
    _check(got, g, steps)


@pytest.mark.parametrize("steps", [5, 12, 19, 30])
@pytest.mark.parametrize("kind", ["equal halves", "equal pairs", "full"])
@pytest.mark.parametrize("rows,cols", [(200, 2048), (300, 2100), (510, 2300)])
def test_two_steps_a_pass(rows, cols, kind, steps):
    """The form of wide matrices, from 256 x 2048 and four times as long as high on, and one of the other side."""
    g = _matrix(kind, rows, cols, rows + steps)
    got = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    if kind != "full":
        _equal_rows(got, kind, rows)
    _check(got, g, steps)


BF16_EXTRA = 2.0 ** -8 + 2.0 ** -9


@pytest.mark.parametrize("steps", [2, 3, 4, 5, 6, 7, 8, 10, 12, 20, 24, 30])
@pytest.mark.parametrize("kind", ["full", "low rank", "rank one", "equal halves", "equal pairs", "four decades"])
@pytest.mark.parametrize("rows,cols", [(130, 300), (200, 2100)])
def test_bf16_steps(rows, cols, kind, steps):
    g = _matrix(kind, rows, cols, rows + steps).bfloat16()
    _check(kan_amd.functional.orthogonalize(g.cuda(), steps=steps), g, steps, BF16_EXTRA)


@pytest.mark.parametrize("steps", [1, 5, 9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_batches_and_layouts_of_large_sides(dtype, steps):
    """Several matrices of scales far apart, one of them zero, row-major, transposed and tall: the same bits."""
    kinds = ["full", "rank one", "equal halves", "four decades"]
    g = torch.stack([_matrix(k, 96, 200, 7) * 10.0 ** (2 * i - 3) for i, k in enumerate(kinds)] + [torch.zeros(96, 200)]).to(dtype)
    base = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    for i in range(4):
        _check(base[i], g[i], steps, BF16_EXTRA if dtype == torch.bfloat16 else 0.0)
    assert (base[4] == 0).all()
    turned = g.cuda().transpose(1, 2).contiguous()
    assert torch.equal(kan_amd.functional.orthogonalize(turned.transpose(1, 2), steps=steps), base)
    assert torch.equal(kan_amd.functional.orthogonalize(turned, steps=steps).transpose(1, 2), base)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [9, 14])
def test_other_coefficients(dtype, steps):
    """The cubic iteration, whose m x m form holds for more steps, and two quintics of other slopes."""
    for co in ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.3465, -1.0598, -0.2868)):
        for kind in ("full", "rank one"):
            g = _matrix(kind, 100, 260, steps).to(dtype)
            got = kan_amd.functional.orthogonalize(g.cuda(), steps=steps, coefficients=co)
            _check(got, g, steps, BF16_EXTRA if dtype == torch.bfloat16 else 0.0, coefficients=co)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_stays_in_its_matrix(dtype):
    g = torch.stack([_matrix("full", 90, 300, s) for s in (1, 2)]).to(dtype)
    alone = kan_amd.functional.orthogonalize(g[1:].cuda())
    g[0, 4, 4] = float("nan")
    both = kan_amd.functional.orthogonalize(g.cuda())
    assert torch.isnan(both[0]).all() and torch.equal(both[1:], alone)


@pytest.mark.parametrize("steps", [0, 1, 7, 9, 10, 12, 18, 20, 30])
@pytest.mark.parametrize("kind", ["full", "low rank", "equal halves", "equal pairs", "four decades"])
@pytest.mark.parametrize("rows,cols", [(64, 512), (33, 900), (40, 41)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_side_steps(rows, cols, kind, steps, dtype):
    """A side of at most 64; the iterate goes on in a run of its own from ten steps of the quintic on."""
    g = _matrix(kind, rows, cols, rows + steps).to(dtype)
    got = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    if kind.startswith("equal") and steps >= 10:
        _equal_rows(got, kind, rows)
    _check(got, g, steps, 1e-6 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0))


@pytest.mark.parametrize("steps", [5, 13])
def test_small_side_batches_and_layouts(steps):
    kinds = ["full", "equal halves", "four decades", "full"]
    g = torch.stack([_matrix(k, 50, 130, 3) * 10.0 ** (3 * i - 4) for i, k in enumerate(kinds)] + [torch.zeros(50, 130)])
    g[3, 2, 2] = float("nan")
    base = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    for i in range(3):
        _check(base[i], g[i], steps, 1e-6)
    assert torch.isnan(base[3]).all() and (base[4] == 0).all()
    turned = g.cuda().transpose(1, 2).contiguous()
    for got in (kan_amd.functional.orthogonalize(turned.transpose(1, 2), steps=steps),
                kan_amd.functional.orthogonalize(turned, steps=steps).transpose(1, 2)):
        assert torch.equal(got.nan_to_num(0.5), base.nan_to_num(0.5))


def test_small_side_other_coefficients():
    for co, steps in (((1.5, -0.5, 0.0), 40), ((1.875, -1.25, 0.375), 25), ((2.3465, -1.0598, -0.2868), 16)):
        g = _matrix("full", 48, 300, steps)
        _check(kan_amd.functional.orthogonalize(g.cuda(), steps=steps, coefficients=co), g, steps, 1e-6, coefficients=co)


@pytest.mark.parametrize("rows,cols", [(80, 2100), (96, 2592), (160, 4032), (192, 2135), (256, 2304), (300, 2500), (512, 4608),
                                       (130, 140), (700, 900)])
def test_no_less_exact_than_plain_products(rows, cols):
    """fp32: at most half as much again as the error of torch's fp32 products, or 1e-6."""
    g = _matrix("full", rows, cols, rows).cuda()
    x = g / (g.norm() + 1e-7)
    for _ in range(5):
        gram = x @ x.t().contiguous()
        x = NS[0] * x + (NS[1] * gram + NS[2] * gram @ gram) @ x
    want = torch.from_numpy(_definition(g.double().cpu().numpy(), 5)).cuda()
    plain = ((x.double() - want).norm() / want.norm()).item()
    got = kan_amd.functional.orthogonalize(g)
    assert ((got.double() - want).norm() / want.norm()).item() <= max(1e-6, 1.5 * plain)


@pytest.mark.parametrize("steps", [1, 3, 5, 8, 12])
@pytest.mark.parametrize("rows,cols", [(70, 150), (300, 2500), (140, 130), (64, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_far_below_eps(rows, cols, dtype, steps):
    """X0 is far below 1 then, and so is the result; its error is held to its own size."""
    g = torch.stack([_matrix("full", rows, cols, i) for i in range(5)])
    g = (g / g.norm(dim=(1, 2), keepdim=True) * torch.tensor([1.0, 1e-8, 1e-11, 1e-15, 1e-22]).view(-1, 1, 1)).to(dtype)
    got = kan_amd.functional.orthogonalize(g.cuda(), steps=steps)
    for i in range(5):
        _check(got[i], g[i], steps, 1e-6 + (BF16_EXTRA if dtype == torch.bfloat16 else 0.0))


def test_a_large_eps():
    g = _matrix("full", 100, 300, 3) * 1e-3
    for eps in (1.0, 1e3):
        _check(kan_amd.functional.orthogonalize(g.cuda(), eps=eps), g, 5, 1e-6, eps=eps)
