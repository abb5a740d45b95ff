"""Log probabilities, entropies, likeliest classes and gradients against the 64-bit definition.

Bounds, with d the largest |l - max| that matters (terms below exp(-30) of the largest are under 2^-43 of a sum) and eps =
2^-24: an exponential is off by (2 |d| + 2) eps relative, of which a sum weighted by exp(-|d|) sees at most a
few (|d| exp(-|d|) <= 0.37 a term, and terms of a sum share it); log Z is off by 8 eps of itself or of the sum's relative error,
16 eps with the order of the sum (log2 and chunks of the fixed order). logp: 16 eps (1 + |logp|). Entropy: 24 eps (1 + H).
A gradient's entry is p times a bracket: p off by (2 |lp| + 18) eps and in bf16 by the
entry's own half step beside it (8 significant bits: 2^-8). In a row that is sure of its largest, 1 - p and log p of
that class are made of exp(-gap), gap being its distance to the next, and carry that term's (2 gap + 2) eps: the
same bound with the gap in lp's place.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import block_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
EPS = 2.0 ** -24
INF = float("inf")


def compare(l, t, top, seed=0):
    """All outputs and the gradient for logits l [rows, classes] and targets t on the host."""
    rows = l.shape[0]
    g = torch.Generator().manual_seed(seed + 1)
    dl, dH = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    leaf = l.cuda().requires_grad_()
    got = f.log_probs(leaf, t.cuda(), top=top)
    logp, H, top_logp, top_idx, lp = orc.log_probs(l.double().numpy(), t.numpy(), top)

    def near(a, want, limit):
        a = a.detach().cpu().double().numpy()
        assert np.array_equal(np.isnan(a), np.isnan(want)) and np.array_equal(np.isinf(a), np.isinf(want))
        ok = np.isfinite(want)
        assert (np.sign(a[~ok & ~np.isnan(want)]) == np.sign(want[~ok & ~np.isnan(want)])).all()
        err = np.abs(np.where(ok, a, 0) - np.where(ok, want, 0))
        assert (err <= np.where(ok, limit, 0)).all(), (err / np.where(ok, limit, 1)).max()

    near(got.logp, logp, 16 * EPS * (1 + np.abs(np.where(np.isfinite(logp), logp, 0))))
    near(got.entropy, H, 24 * EPS * (1 + np.abs(H)))
    if top:
        assert np.array_equal(got.top_indices.cpu().numpy(), top_idx)
        near(got.top_logp, top_logp, 16 * EPS * (1 + np.abs(np.where(np.isfinite(top_logp), top_logp, 0))))
    else:
        assert got.top_logp is None and got.top_indices is None
    d, = torch.autograd.grad((got.logp, got.entropy), leaf, (dl.cuda(), dH.cuda()))
    assert d.dtype == l.dtype
    want, size = orc.log_probs_backward(l.double().numpy(), t.numpy(), dl.double().numpy(), dH.double().numpy())
    two = np.sort(np.where(np.isfinite(lp), lp, -np.inf), 1)[:, -2:]
    gap = two[:, -1] - two[:, 0]
    gap = np.where(np.isfinite(gap), gap, 0)[:, None]
    off = 2 * np.maximum(np.abs(np.where(np.isfinite(lp), lp, 0)), gap) + 18
    near(d, want, size * off * EPS + (2.0 ** -8 if l.dtype == torch.bfloat16 else 0) * np.abs(want) * (1 + off * EPS) + 1e-37)
    with torch.no_grad():
        again = f.log_probs(l.cuda(), t.cuda(), top=top)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0))
    return got


def logits(rows, classes, dtype, seed, grid=True):
    g = torch.Generator().manual_seed(seed)
    l = 3 * torch.randn(rows, classes, generator=g)
    return (torch.round(l * 4) / 4 if grid else l).to(dtype), torch.randint(0, classes, (rows,), generator=g)


@pytest.mark.parametrize("classes", [1, 2, 3, 7, 8, 10, 33, 63, 64, 65, 100, 128, 129, 250, 256, 300, 512, 513, 1000, 1023, 2048,
                                     2049, 4100, 8191, 10000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_classes(classes, dtype):
    for rows, top, grid in ((5, min(5, classes), True), (2, min(64, classes), False), (1, 0, False)):
        l, t = logits(rows, classes, dtype, classes + rows, grid)
        compare(l, t, top)


@pytest.mark.parametrize("rows", [1, 3, 4, 31, 256, 1001])
@pytest.mark.parametrize("classes", [10, 100, 600])
def test_rows(rows, classes):
    l, t = logits(rows, classes, torch.float32, rows)
    t[::3] = -100
    t[1::5] = classes
    compare(l, t, 3)


@pytest.mark.parametrize("classes", [20, 300, 3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_ties_and_rows_of_nothing(classes, dtype):
    l, t = logits(14, classes, dtype, 3)
    low = torch.finfo(dtype).min
    l[0] = -INF                      # nothing left
    l[1] = -INF
    l[1, classes - 1] = -2.0         # one class
    t[1] = classes - 1
    l[2, ::2] = -INF
    t[2] = 0                         # the target itself has no probability
    l[3] = low                       # the lowest value everywhere: uniform
    l[4, 1:] = low
    l[4, 0] = 1.0
    t[4] = 0
    l[5] = 0.0                       # all equal: the lowest indices
    l[6] = -l[6].abs()
    l[6, 5] = 0.0
    l[6, 3] = -0.0                   # equal to 0
    l[7] = -INF
    l[7, 4:7] = 1.5
    l[8, 9] = float("nan")
    l[9, 9] = INF
    l[10] = 30.0 * l[10]             # sure rows
    l[11] = torch.finfo(dtype).max / 2
    l[11, 2] = torch.finfo(dtype).max
    t[12] = -1
    l[13] = float("nan")
    for top in (0, 7, 12):
        compare(l, t, top)


@pytest.mark.parametrize("classes", [2050, 3001, 4088, 4095, 4096, 4097, 4104])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_where_rows_leave_the_registers(classes, dtype):
    for rows, top in ((1, 64), (7, 10), (530, 3)):
        l, t = logits(rows, classes, dtype, classes + rows)
        l[0, classes - 9:] = 20.0  # equal ones in a row's last chunks
        l[rows - 1] = torch.sort(l[rows - 1]).values
        compare(l, t, top)


def test_sure_rows_keep_their_relative_precision():
    """exp(-d) for d up to 80 beside the largest: log p and entropy to a few half steps of themselves."""
    for classes in (16, 900, 5000):
        l = torch.full((8, classes), -200.0)
        l[:, 3] = 0.0
        l[:, 11] = -10.0 * torch.arange(1, 9)
        t = torch.full((8,), 3)
        got = compare(l, t, 2)
        d = 10.0 * np.arange(1, 9)
        rest = np.exp(-d) / (1 + np.exp(-d))
        assert (np.abs(got.logp.detach().cpu().numpy() / -np.log1p(np.exp(-d)) - 1) <= (2 * d + 20) * EPS).all()
        H = np.log1p(np.exp(-d)) + rest * d
        assert (np.abs(got.entropy.detach().cpu().numpy() / H - 1) <= (4 * d + 40) * EPS).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows(dtype):
    for classes, rows in ((131072, 1), (131071, 2), (50001, 3)):
        for grid in (True, False):
            l, t = logits(rows, classes, dtype, classes, grid)
            compare(l, t, 20)
    l, t = logits(2, 70000, dtype, 8)
    l = torch.sort(l, dim=1).values  # the largest all in one place
    compare(l, t, 64)
    compare(l.flip(1), t, 64)


def test_layouts_and_shapes():
    l = torch.randn(4, 6, 40, device="cuda")
    t = torch.randint(0, 30, (4, 6), device="cuda")
    for a, b in ((l, t), (l[..., 1:38], t), (l.transpose(0, 1), t.t()), (l[:, 2], t[:, 2]), (l[0, 0], t[0, 0]), (l[:0], t[:0]),
                 (l[:1].expand(4, 6, 40), t), (l.bfloat16()[..., 3:], t)):
        def call(a, b):
            leaf = a.detach().requires_grad_()
            got = f.log_probs(leaf, b, top=3)
            assert got.logp.shape == got.entropy.shape == b.shape and got.top_indices.shape == b.shape + (3,)
            up = torch.ones((), device="cuda").expand(b.shape)
            return [*got, *torch.autograd.grad((got.logp, got.entropy), leaf, (up, up))]
        for u, v in zip(call(a, b), call(a.contiguous().clone(), b.contiguous().clone())):
            assert torch.equal(u, v)


def test_one_upstream_gradient_and_cross_entropy():
    l, t = logits(50, 30, torch.float32, 1, False)
    for keep in ("logp", "entropy"):
        leaf = l.cuda().requires_grad_()
        got = f.log_probs(leaf, t.cuda())
        a, = torch.autograd.grad(getattr(got, keep).sum(), leaf)
        leaf2 = l.cuda().requires_grad_()
        got2 = f.log_probs(leaf2, t.cuda())
        other = got2.entropy if keep == "logp" else got2.logp
        b, = torch.autograd.grad(getattr(got2, keep).sum() + 0 * other.sum(), leaf2)
        assert torch.equal(a, b)
    leaf = l.cuda().requires_grad_()
    loss = -f.log_probs(leaf, t.cuda()).logp.mean()
    g, = torch.autograd.grad(loss, leaf)
    ref = l.double().requires_grad_()
    want = torch.nn.functional.cross_entropy(ref, t)
    gw, = torch.autograd.grad(want, ref)
    assert abs(loss.item() - want.item()) <= 32 * EPS * (1 + want.item())
    assert (g.cpu().double() - gw).abs().max() <= 64 * EPS / 50


def test_changed_inputs_are_refused():
    l, t = logits(4, 9, torch.float32, 1)
    leaf = l.cuda().requires_grad_()
    t = t.cuda()
    got = f.log_probs(leaf, t)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(got.logp.sum(), leaf, create_graph=True)
    got = f.log_probs(leaf, t)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(got.logp.sum(), leaf)
