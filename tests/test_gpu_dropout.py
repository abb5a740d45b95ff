"""Dropout's mask against the generator's definition, and its results to the bit: each is one product and one rounding."""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import block_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def expected(x, keep, p):
    factor = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32)
    return torch.where(torch.from_numpy(keep), x.float() * factor, 0.0).to(x.dtype)


@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 7), (3, 8), (5, 9), (256, 10), (33, 65), (2, 784), (7, 1029), (1, 5000),
                                      (1000, 24), (3, 16385)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 1e-4, 0.1, 0.5, 0.9999, 1.0])
def test_mask_and_gradient(rows, dim, dtype, p):
    x = (torch.randn(rows, dim, generator=torch.Generator().manual_seed(dim)) + 3).to(dtype)
    dy = torch.randn(rows, dim, generator=torch.Generator().manual_seed(dim + 1)).to(dtype)
    for seed, call, as_int in ((2 ** 63 + 12345, 0, True), (-5, 2 ** 33 + 7, False)):
        state = seed if as_int else torch.tensor([seed, 3], device="cuda")
        keep = orc.keep_mask(seed, call + (0 if as_int else 3), rows, dim, p)
        leaf = x.cuda().requires_grad_()
        y = f.dropout(leaf, p, state, call)
        assert torch.equal(y.cpu(), expected(x, keep, p))
        if not as_int:
            state.add_(100)  # the gradient belongs to the state as the forward read it
        dx, = torch.autograd.grad(y, leaf, dy.cuda())
        assert torch.equal(dx.cpu(), expected(dy, keep, p))


def test_the_low_halves_decide():
    """Thresholds whose high half is met: 2^-16 of the elements need the second stream."""
    x = torch.ones(512, 1024)
    for p in (3.0 / 2 ** 17, 0.5 + 2.0 ** -18, 1.0 - 2.0 ** -32, 2.0 ** -32, 0.3):
        keep = orc.keep_mask(31, 8, 512, 1024, p)
        y = f.dropout(x.cuda(), p, 31, 8)
        assert np.array_equal((y != 0).cpu().numpy(), keep)


def test_values_that_are_dropped_do_not_matter():
    x = torch.full((4, 96), float("nan"), device="cuda")
    x[:, ::2] = float("inf")
    keep = orc.keep_mask(3, 0, 4, 96, 0.5)
    y = f.dropout(x, 0.5, 3).cpu()
    assert torch.equal(y[~torch.from_numpy(keep)], torch.zeros(int((~keep).sum())))
    assert not torch.isfinite(y[torch.from_numpy(keep)]).any()


def test_layouts_and_shapes():
    wide = torch.randn(6, 5, 50, device="cuda")
    for x in (wide, wide[0, 0], wide[:, :, 1:9], wide.transpose(0, 1), wide[:, 2], wide[:1, :1].expand(6, 5, 50), wide[:0],
              wide[..., :0]):
        got = f.dropout(x, 0.4, 11)
        assert got.shape == x.shape and torch.equal(got, f.dropout(x.contiguous(), 0.4, 11))
        leaf = x.detach().requires_grad_()
        y = f.dropout(leaf, 0.4, 11)
        g, = torch.autograd.grad(y, leaf, torch.ones(1, device="cuda").expand(y.shape))
        assert torch.equal(g, f.dropout(torch.ones_like(x), 0.4, 11))


def test_the_residual_draws_the_same_mask():
    x = torch.zeros(37, 130, device="cuda")
    y = torch.randn_like(x)
    state = torch.tensor([99, 4], device="cuda")
    out = f.residual_norm(x, y, dropout=0.3, dropout_state=state, dropout_call=6)
    assert torch.equal(out, f.dropout(y, 0.3, state, 6)) and torch.equal(out, f.dropout(y, 0.3, 99, 10))


def test_refusals():
    x = torch.zeros(2, 4, device="cuda")
    for state in (None, 1.5):
        with pytest.raises(ValueError, match="state"):
            f.dropout(x, 0.5, state)
    for state in (torch.zeros(2, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int64),
                  torch.zeros(2, dtype=torch.int64), torch.zeros(4, device="cuda", dtype=torch.int64)[::2]):
        with pytest.raises(RuntimeError, match="state"):
            f.dropout(x, 0.5, state)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            f.dropout(x, p, 1)
    with pytest.raises(ValueError, match="call"):
        f.dropout(x, 0.5, 1, -1)
    leaf = x.requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(f.dropout(leaf, 0.5, 1).sum(), leaf, create_graph=True)
