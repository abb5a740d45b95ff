"""The residual block, dropout and log probabilities past 2^31 elements: what lies beyond gives the same as the same
values in small tensors."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def test_residual_rows_past_32_bits():
    rows, dim, tail = 4300000, 512, 600
    x, y = (torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert x.numel() > 2 ** 31
    kw = {k: torch.randn(dim, device="cuda") for k in ("post_weight", "gate", "next_weight")}
    got = []
    for a, b in ((x, y), (x[-tail:].clone(), y[-tail:].clone())):
        a.requires_grad_(), b.requires_grad_()
        out, h = f.residual_norm(a, b, norm="layer", **kw)
        up = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(out.shape)
        dx, dy = torch.autograd.grad((out, h), (a, b), (out.detach(), up))
        got.append([t[-tail:].clone() for t in (out.detach(), h.detach(), dx, dy)])
        del out, h, dx, dy
    for u, v in zip(*got):
        assert torch.equal(u, v)


def test_residual_parameters_of_rows_past_32_bits():
    """The sums over rows of a tensor whose last rows alone have an upstream gradient: the sums of those rows, in
    another order: each of two sums of 600 terms is off by at most 600 half steps of the sum of their absolute values."""
    rows, dim, tail = 4300000, 512, 600
    x = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(dim, device="cuda", requires_grad=True)
    up = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    up[-tail:].normal_()
    a, = torch.autograd.grad(f.row_norm(x, w), w, up)
    b, = torch.autograd.grad(f.row_norm(x[-tail:], w), w, up[-tail:])
    size, = torch.autograd.grad(f.row_norm(x[-tail:].abs(), w), w, up[-tail:].abs())
    assert ((a - b).abs() <= 2 * tail * 2.0 ** -24 * size).all()


def test_dropout_past_32_bits():
    x = torch.ones(4300000, 512, device="cuda", dtype=torch.bfloat16)
    a = f.dropout(x, 0.3, 9, 4)
    # the block's kernel draws the same numbers from rows and columns of its own counting
    b = f.residual_norm(torch.zeros_like(x), x, dropout=0.3, dropout_state=9, dropout_call=4)
    assert torch.equal(a, b)
    kept = (a[-5000:] != 0).double().mean().item()
    assert abs(kept - 0.7) <= 5 * (0.21 / (5000 * 512)) ** 0.5  # standard deviations of a share
    del a, b, x
    x = torch.ones(2, 2 ** 30 + 8, device="cuda", dtype=torch.bfloat16)
    y = f.dropout(x, 0.3, 9)
    kept = (y[1, -(1 << 20):] != 0).double().mean().item()
    assert abs(kept - 0.7) <= 5 * (0.21 / (1 << 20)) ** 0.5
    assert set(y[1, -1000:].tolist()) == {0.0, torch.tensor(1 / 0.7).bfloat16().item()}


def test_logits_past_32_bits():
    rows, classes, tail = 43000, 50001, 1000
    l = torch.randn(rows, classes, device="cuda", dtype=torch.bfloat16)
    assert l.numel() > 2 ** 31 and (rows - tail) * classes % 8 == 0  # the tail's rows lie as in its copy
    t = torch.randint(0, classes, (rows,), device="cuda")
    dl = torch.randn(rows, device="cuda")
    got = []
    for a, b, d in ((l, t, dl), (l[-tail:].clone(), t[-tail:].clone(), dl[-tail:])):
        a.requires_grad_()
        p = f.log_probs(a, b, top=5)
        g, = torch.autograd.grad((p.logp, p.entropy), a, (d, d))
        got.append([v[-tail:].detach().clone() for v in (*p, g)])
        del p, g
    for u, v in zip(*got):
        assert torch.equal(u, v)
