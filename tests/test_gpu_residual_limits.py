"""Residual blocks of rows whose mean over its root mean square passes fp32's range.

Rows of one value 2^k whose mean is exact (the partial sums are multiples of 2^k below 2^24 of them, and the widths are those
whose rounded reciprocal gives back 1): the values less their mean are 0, so norms give their biases exactly and gradients
are sums over eps alone. Places past a row's end have no part in that, although mean / sqrt(eps) overflows.
"""
import numpy as np
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional
DIMS = [9, 10, 32, 50, 64, 100, 300, 520, 1000, 1029, 2050, 5000, 6001, 9000]


def exact_mean(dim):
    return np.float32(dim) * (np.float32(1) / np.float32(dim)) == 1


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_one_large_value(dim, dtype):
    """out = x + scale gate b (lost beside x), h = b', and with e^ = 0 the gradients r (g - mean g), chained.

    Each difference from a row's mean is off by at most (48 + dim / 256) half steps of its terms, as the other tests of
    these operators have it, and dy chains two of them."""
    assert exact_mean(dim)
    rows, eps, big, scale = 5, 1e-20, 2.0 ** 100, 0.5
    g = torch.Generator().manual_seed(dim)
    draw = lambda *s: torch.randn(*s, generator=g).to(dtype)
    w1, b1, w2, b2, gate = (draw(dim) for _ in range(5))
    dout, dh = draw(rows, dim), draw(rows, dim)
    x = torch.full((rows, dim), big, dtype=dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, x, gate, w1, b1, w2, b2)]
    out, h = f.residual_norm(leaves[0], leaves[1], norm="layer", eps=eps, scale=scale, gate=leaves[2], post_weight=leaves[3],
                             post_bias=leaves[4], next_weight=leaves[5], next_bias=leaves[6])
    assert torch.equal(out.detach().cpu(), x) and torch.equal(h.detach().cpu(), b2.expand(rows, dim))
    dx, dy, dgate, dw1, db1, dw2, db2 = (t.cpu().double() for t in torch.autograd.grad((out, h), leaves, (dout.cuda(), dh.cuda())))
    r = 1.0 / np.sqrt(eps)
    steps = (48 + dim / 256) * 2.0 ** -24

    def centred(v, mag):
        return r * (v - v.mean(-1, keepdim=True)), r * (mag + mag.mean(-1, keepdim=True))

    def near(name, got, want, mag, k):
        limit = k * steps * mag + (torch.finfo(dtype).eps / 2) * want.abs() * (1 + k * steps) + 1e-37
        worst = ((got - want).abs() / limit).max().item()
        assert worst <= 1.0, f"{name}: {worst:.2f} of its bound"

    w1, b1, w2, gate, dout, dh = (t.double() for t in (w1, b1, w2, gate, dout, dh))
    v, mag = centred(dh * w2, (dh * w2).abs())
    v, mag = dout + v, dout.abs() + mag
    near("dx", dx, v, mag, 1)
    near("dgate", dgate, (scale * v * b1).sum(0), (scale * mag * b1.abs()).sum(0), 1 + rows)
    v, mag = scale * gate * v, scale * gate.abs() * mag
    near("dpost_bias", db1, v.sum(0), mag.sum(0), 1 + rows)
    near("dy", dy, *centred(v * w1, mag * w1.abs()), 2)
    near("dnext_bias", db2, dh.sum(0), dh.abs().sum(0), 1 + rows)
    assert not dw1.any() and not dw2.any()

