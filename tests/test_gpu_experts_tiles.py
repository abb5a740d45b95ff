"""The experts' products of many output tiles: wide and narrow tiles, tiles that are not split along k, whole rounds of
them with and without a rest, and plans of more slots than one pass of their blocks takes.

The reference is the definition in 64-bit torch products.  Bounds as in test_gpu_experts.py: fp32 5e-6, bf16 5e-3 of the
result's norm.  `launches` restates how the library shares out its tiles, so that each case says which form it runs.
"""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 5e-6, torch.bfloat16: 5e-3}
ROUND, SPLITS = 64, 8  # tiles an XCD has in flight; the most parts of a split tile


def _ceil(a, b):
    return -(-a // b)


def _rounds(tiles):
    n = _ceil(tiles, 8)
    rest = n % ROUND
    return n // ROUND + (1 / min(SPLITS, ROUND // rest) if rest else 0)


def _share(tiles):
    """(whole rounds, parts of the rest's tiles; 1: not split, 0: no rest) of an XCD with a full share."""
    n = _ceil(tiles, 8)
    rest = n % ROUND
    return n // ROUND, min(SPLITS, ROUND // rest) if rest else 0


def launches(idx, experts, in_dim, out, degree, dtype):
    """(width, (rounds, parts)) of the forward and (rounds, parts) of dx."""
    slots = idx.numel()
    at_most = _ceil(slots, 128) + min(experts, slots)
    narrow, wide = 1.1 * _rounds(at_most * _ceil(out, 128)), 2 * _rounds(at_most * _ceil(out, 256))
    width = 128 if (dtype == torch.float32 and degree > 8) or narrow < wide else 256
    tiles = int(sum(_ceil(int(n), 128) for n in torch.bincount(idx.reshape(-1), minlength=experts)))
    return (width, _share(tiles * _ceil(out, width))), _share(tiles * _ceil(_ceil(in_dim, 32) * 32, 64))


def _basis(x, degree):
    """T_0..T_degree of tanh x and their derivatives in x, [rows, in, degree + 1]."""
    t = torch.tanh(x)
    T, U = [torch.ones_like(t), t], [torch.ones_like(t), 2 * t]
    for _ in range(degree - 1):
        T.append(2 * t * T[-1] - T[-2])
        U.append(2 * t * U[-1] - U[-2])
    slope = [torch.zeros_like(t)] + [d * U[d - 1] for d in range(1, degree + 1)]
    return torch.stack(T, -1), torch.stack(slope, -1) * (1 - t * t)[..., None]


def _reference(x, c, idx, w, dy):
    experts, in_dim, out, dd = c.shape
    y = torch.zeros(x.shape[0], out, dtype=torch.float64, device=x.device)
    dx, dc, dw = torch.zeros_like(x), torch.zeros_like(c), torch.zeros_like(w)
    for e in range(experts):
        rows, j = torch.nonzero(idx == e, as_tuple=True)
        T, slope = _basis(x[rows], dd - 1)
        C = c[e].permute(0, 2, 1).reshape(in_dim * dd, out)
        z = T.flatten(1) @ C
        y.index_add_(0, rows, w[rows, j][:, None] * z)
        dw[rows, j] = (z * dy[rows]).sum(1)
        g = w[rows, j][:, None] * dy[rows]
        dc[e] = (T.flatten(1).t().contiguous() @ g).reshape(in_dim, dd, out).permute(0, 2, 1)
        back = (g @ C.t().contiguous()).reshape(len(rows), in_dim, dd)
        dx.index_add_(0, rows, (back * slope).sum(2))
    return y, dx, dc, dw


def _case(rows, in_dim, out, degree, experts, top_k, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, in_dim, generator=g, device="cuda").to(dtype)
    c = (torch.randn(experts, in_dim, out, degree + 1, generator=g, device="cuda") / (in_dim * (degree + 1))).to(dtype)
    idx = (torch.rand(rows, experts, generator=g, device="cuda") + torch.rand(experts, generator=g, device="cuda")).topk(top_k, 1)[1]
    w = torch.rand(rows, top_k, generator=g, device="cuda") + 0.2
    dy = torch.randn(rows, out, generator=g, device="cuda").to(dtype)
    return x, c, idx, w, dy


def _compare(x, c, idx, w, dy, dtype):
    args = [v.clone().requires_grad_() for v in (x, c, w)]
    y = kan_amd.functional.kan_experts(args[0], args[1], idx, args[2])
    got = (y.detach(),) + torch.autograd.grad(y, args, dy)
    want = _reference(x.double(), c.double(), idx, w.double(), dy.double())
    with torch.no_grad():
        got += (kan_amd.functional.kan_experts(x, c, idx, w),)
    for name, a, b in zip(("y", "dx", "dcoeffs", "dweights", "y without a backward"), got, want + want[:1]):
        assert torch.isfinite(a).all(), name
        assert (a.double() - b).norm() <= TOL[dtype] * b.norm(), name


F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("rows,in_dim,out,degree,experts,top_k,dtype,forward,dx", [
    # wide tiles: unsplit, one whole round, a round and a rest, all split
    (8000, 40, 1000, 8, 3, 2, F32, (256, (1, 0)), (0, 4)),
    (8000, 40, 1000, 8, 3, 2, BF16, (256, (1, 0)), (0, 4)),
    (8800, 36, 1013, 4, 3, 2, F32, (256, (1, 8)), (0, 3)),
    (8800, 36, 1013, 4, 3, 2, BF16, (256, (1, 8)), (0, 3)),
    (6500, 70, 1021, 3, 3, 2, F32, (256, (0, 1)), (0, 2)),
    (6500, 70, 1021, 3, 3, 2, BF16, (256, (0, 1)), (0, 2)),
    (8000, 33, 1000, 16, 3, 2, BF16, (256, (1, 0)), (0, 4)),
    # narrow tiles: a round and a rest, and an unsplit rest on two planes of 16 degrees, odd sizes
    (8000, 150, 600, 3, 4, 2, F32, (128, (1, 4)), (0, 1)),
    (8000, 150, 600, 3, 4, 2, BF16, (128, (1, 4)), (0, 1)),
    (8000, 33, 1000, 12, 3, 2, F32, (128, (1, 1)), (0, 4)),
    (8800, 64, 300, 16, 5, 2, F32, (128, (0, 1)), (0, 3)),
    # dx: whole rounds and a rest, several groups of 16 tiles by several columns
    (9001, 300, 130, 4, 5, 2, F32, (256, (0, 3)), (1, 2)),
    (9001, 300, 130, 4, 5, 2, BF16, (256, (0, 3)), (1, 2)),
    (4300, 500, 72, 5, 40, 3, F32, (128, (0, 4)), (1, 1)),
])
def test_many_tiles(rows, in_dim, out, degree, experts, top_k, dtype, forward, dx):
    x, c, idx, w, dy = _case(rows, in_dim, out, degree, experts, top_k, dtype, rows + out)
    assert launches(idx.cpu(), experts, in_dim, out, degree, dtype) == (forward, dx)
    _compare(x, c, idx, w, dy, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_plan_of_many_slots(dtype):
    """300000 slots: a block of the plan places more than one chunk of 1024."""
    _compare(*_case(150000, 4, 5, 1, 7, 2, dtype, 1), dtype)


def test_dropped_slots_of_many_tiles():
    x, c, idx, w, dy = _case(8000, 150, 600, 3, 4, 2, F32, 5)
    idx[::3, 1] = -1
    idx[idx == 2] = 99
    _compare(x, c, idx, w, dy, F32)
