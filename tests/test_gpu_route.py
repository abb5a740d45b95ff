"""Routing to experts against the 64-bit definition: choices, weights and gradients.

Bounds: a weight is a quotient of scores, each a few fp32 roundings of an
exponential (2 ulp), a sum and a division: under 16 half-ulps, 1e-6 relative to
the largest weight.  A gradient entry is a product of such factors with dw over
the chosen sum, which cancels by the dw's mean: 4e-6 relative to the row's largest
entry; rounding to bf16 adds 2^-9.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

CASES = [
    # rows, experts, top_k, score, groups, top_groups, bias, dtype
    (1, 8, 2, "softmax", 1, 1, False, torch.float32),
    (1, 1, 1, "softmax", 1, 1, False, torch.float32),
    (5, 2, 2, "sigmoid", 1, 1, True, torch.float32),
    (7, 64, 8, "softmax", 1, 1, True, torch.float32),
    (130, 60, 6, "softmax", 1, 1, False, torch.bfloat16),
    (33, 65, 5, "sigmoid", 5, 2, False, torch.float32),
    (64, 256, 8, "sigmoid", 8, 4, True, torch.float32),
    (19, 256, 6, "softmax", 32, 3, True, torch.bfloat16),
    (9, 510, 17, "softmax", 3, 2, False, torch.float32),
    (3, 512, 64, "sigmoid", 64, 8, True, torch.float32),
    (4, 64, 3, "softmax", 64, 5, False, torch.float32),
    (1001, 16, 4, "sigmoid", 4, 2, True, torch.bfloat16),
]


def _inputs(rows, experts, dtype, seed, ties=True):
    """Logits on a grid of 1/8 (exact in bf16, many equal ones), or spread out."""
    g = torch.Generator().manual_seed(seed)
    l = 2.0 * torch.randn(rows, experts, generator=g)
    if ties:
        l = torch.round(l * 8) / 8
    return l.to(dtype)


def _check_choice(l, idx, w, kw, top_k):
    want_w, want = orc.route(l.double().numpy(), top_k, **kw)
    assert np.array_equal(idx.cpu().numpy(), want)
    assert np.abs(w.cpu().numpy() - want_w).max() <= 1e-6 * max(1.0, want_w.max())


@pytest.mark.parametrize("rows,experts,top_k,score,groups,top_groups,bias,dtype", CASES)
def test_choice_weights_and_gradient(rows, experts, top_k, score, groups, top_groups, bias, dtype):
    for seed, renormalize, scale in ((1, True, 1.0), (2, False, 2.5)):
        l = _inputs(rows, experts, dtype, seed)
        # biases on a grid that keeps unequal keys apart by far more than an fp32 rounding
        b = (torch.randint(-3, 4, (experts,), generator=torch.Generator().manual_seed(seed)).double()
             * 0.171).float() if bias else None
        kw = dict(score=score, bias=None if b is None else b.numpy(), groups=groups, top_groups=top_groups,
                  renormalize=renormalize, scale=scale)
        ld = l.cuda().requires_grad_()
        w, idx = kan_amd.functional.route(ld, top_k, **{**kw, "bias": None if b is None else b.cuda()})
        _check_choice(l, idx, w.detach(), kw, top_k)
        dw = torch.randn(rows, top_k, generator=torch.Generator().manual_seed(seed + 7))
        got, = torch.autograd.grad(w, ld, dw.cuda())
        assert got.dtype == dtype
        want = orc.route_backward(l.double().numpy(), idx.cpu().numpy(), dw.numpy(), score, renormalize, scale)
        tol = 4e-6 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol * np.abs(want).max() + 1e-12


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_and_empty_rows(score):
    l = _inputs(12, 24, torch.float32, 5)
    l[0] = -float("inf")                       # nothing to choose
    l[1, 3:] = -float("inf")                   # fewer experts than slots
    l[2, ::2] = float("nan")
    l[3] = torch.finfo(torch.float32).min      # the lowest value everywhere: still eligible
    l[4, 1:] = torch.finfo(torch.float32).min
    l[5, :12] = -float("inf")                  # whole groups gone
    l[6] = 80.0                                # all equal, sigmoid saturated
    for groups, top_groups in ((1, 1), (4, 2)):
        kw = dict(score=score, groups=groups, top_groups=top_groups)
        ld = l.cuda().requires_grad_()
        w, idx = kan_amd.functional.route(ld, 5, **kw)
        _check_choice(l, idx, w.detach(), kw, 5)
        assert (idx[0] == -1).all() and (w[0] == 0).all()
        got, = torch.autograd.grad(w, ld, torch.ones_like(w) + torch.arange(5.0, device="cuda"))
        assert torch.isfinite(got).all()
        assert (got[0] == 0).all() and (got[1, 3:] == 0).all()


def test_strided_logits_other_stream_and_empty():
    l = _inputs(40, 96, torch.float32, 9)
    wide = torch.full((40, 200), 100.0)
    wide[:, 50:146] = l
    view = wide.cuda()[:, 50:146]
    base = kan_amd.functional.route(l.cuda(), 4)
    for got in (kan_amd.functional.route(view, 4), kan_amd.functional.route(l.t().contiguous().cuda().t(), 4)):
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kan_amd.functional.route(view, 4)
    side.synchronize()
    assert torch.equal(got[1], base[1])
    w, idx = kan_amd.functional.route(torch.empty(0, 8, device="cuda", requires_grad=True), 2)
    assert w.shape == (0, 2) and idx.shape == (0, 2)
    w.sum().backward()
    same = kan_amd.functional.route(torch.zeros(1, 7, device="cuda").expand(6, 7), 3)
    assert same[1].tolist() == [[0, 1, 2]] * 6


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinite_logit_takes_its_limit(score):
    l = _inputs(3, 70, torch.float32, 21)
    l[0, 66] = float("inf")
    l[1, 5] = float("inf")
    l[1, 6] = -float("inf")
    kw = dict(score=score, renormalize=False)
    ld = l.cuda().requires_grad_()
    w, idx = kan_amd.functional.route(ld, 3, **kw)
    assert idx[0, 0] == 66 and idx[1, 0] == 5 and (w[:2, 0] == 1).all()
    _check_choice(l.clamp(max=torch.finfo(torch.float32).max), idx, w.detach(), kw, 3)
    got, = torch.autograd.grad(w.sum(), ld)
    assert torch.isfinite(got).all()


def test_indices_changed_before_the_backward_are_refused():
    ld = _inputs(4, 9, torch.float32, 2).cuda().requires_grad_()
    w, idx = kan_amd.functional.route(ld, 2)
    idx[0, 0] = -1
    with pytest.raises(RuntimeError, match="modified in place"):
        w.sum().backward()


def test_second_derivative_is_refused():
    ld = _inputs(4, 9, torch.float32, 2).cuda().requires_grad_()
    w, _ = kan_amd.functional.route(ld, 2)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(w.square().sum(), ld, create_graph=True)
