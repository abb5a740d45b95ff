"""Newton-Schulz orthogonalisation and Muon's step against the definition in 64 bits.

Bound in fp32: five steps, each a chain of three products whose entries carry
about 2^-22 (operands) and sqrt(K) 2^-24 (sums) of the product of norms.  Five steps
take small singular values up by 3.4^5, signal and error alike, so the result's
relative error is a few times 2^-22 sqrt(steps): 1e-5 with a margin of about 5
(plain fp32 products measure 1-3e-6).  bf16 results add their rounding:
half an ulp, at most 2^-8 of a value (8 significant bits).
"""
import math

import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

FP32_TOL = 1e-5
BF16_TOL = 1e-5 + 2.0 ** -8


def _gradient(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(rows, cols) // 32)
    strong = torch.randn(rows, r, generator=g) @ torch.randn(r, cols, generator=g) / math.sqrt(r)
    return 1e-3 * (strong + 0.3 * torch.randn(rows, cols, generator=g))


def _rel(got, want):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    return np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 300), (5, 3), (16, 16), (32, 33), (64, 3920), (65, 64),
                                       (127, 129), (128, 128), (130, 1000), (300, 3000), (900, 500), (700, 20),
                                       (257, 2305)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize(rows, cols, dtype):
    g = _gradient(rows, cols, rows + cols).to(dtype)
    got = kan_amd.functional.orthogonalize(g.cuda())
    assert got.dtype == dtype and got.shape == g.shape
    want = orc.orthogonalize(g.double().numpy())
    assert _rel(got, want) <= (FP32_TOL if dtype == torch.float32 else BF16_TOL)


def test_batches_layouts_and_steps():
    gs = [_gradient(70, 150, s) * 10.0 ** (3 * s - 6) for s in range(5)]  # scales 1e-9 .. 1e3
    g = torch.stack(gs).cuda()
    base = kan_amd.functional.orthogonalize(g, eps=1e-20)
    for k in range(5):
        assert _rel(base[k], orc.orthogonalize(gs[k].double().numpy(), eps=1e-20)) <= FP32_TOL
    # the same matrices as transposed views, strided slices and more batch dimensions: the same bits
    t = g.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kan_amd.functional.orthogonalize(t, eps=1e-20), base)
    wide = torch.zeros(5, 70, 200, device="cuda")
    wide[:, :, 20:170] = g
    assert torch.equal(kan_amd.functional.orthogonalize(wide[:, :, 20:170], eps=1e-20), base)
    more = g.reshape(5, 1, 70, 150)
    assert torch.equal(kan_amd.functional.orthogonalize(more, eps=1e-20), base.reshape(5, 1, 70, 150))
    # tall is the transpose of wide
    tall = kan_amd.functional.orthogonalize(g.transpose(1, 2).contiguous(), eps=1e-20)
    assert torch.equal(tall.transpose(1, 2), base)
    for steps in (0, 1, 2, 9):
        got = kan_amd.functional.orthogonalize(g[2], steps=steps)
        assert _rel(got, orc.orthogonalize(gs[2].double().numpy(), steps=steps)) <= FP32_TOL
    gentle = (1.5, -0.5, 0.0)  # the cubic iteration
    got = kan_amd.functional.orthogonalize(g[2], steps=7, coefficients=gentle)
    assert _rel(got, orc.orthogonalize(gs[2].double().numpy(), 7, gentle)) <= FP32_TOL
    assert kan_amd.functional.orthogonalize(torch.empty(0, 3, 4, device="cuda")).shape == (0, 3, 4)


def test_degenerate_matrices():
    z = torch.zeros(2, 40, 60, device="cuda")
    assert (kan_amd.functional.orthogonalize(z) == 0).all()
    z[1, 3, 5] = -7.0  # one entry: rank 1, the whole norm in one place
    got = kan_amd.functional.orthogonalize(z)
    assert (got[0] == 0).all()
    assert _rel(got[1], orc.orthogonalize(z[1].double().cpu().numpy())) <= FP32_TOL
    bad = _gradient(40, 60, 1)
    bad[4, 4] = float("nan")
    both = torch.stack([bad, _gradient(40, 60, 2)]).cuda()
    got = kan_amd.functional.orthogonalize(both)  # NaN stays in its own matrix
    assert torch.isnan(got[0]).all()
    assert _rel(got[1], orc.orthogonalize(both[1].double().cpu().numpy())) <= FP32_TOL


def test_repeats_bit_for_bit_and_on_another_stream():
    g = _gradient(200, 1500, 3).cuda()
    base = kan_amd.functional.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [kan_amd.functional.orthogonalize(g) for _ in range(3)]
    side.synchronize()
    for v in got:
        assert torch.equal(v, base)


@pytest.mark.parametrize("shape", [(64, 48), (48, 200), (20, 33, 5), (7, 90, 3), (12, 10, 1), (3, 40, 32, 9)])
def test_muon_step(shape):
    gen = torch.Generator().manual_seed(len(shape))
    p = torch.randn(*shape, generator=gen) * 0.01
    g = torch.randn(*shape, generator=gen) * 1e-3
    buf = torch.randn(*shape, generator=gen) * 1e-3
    for nesterov in (True, False):
        pd, bd = p.cuda(), buf.cuda()
        version = pd._version
        kan_amd.optim.muon_step_(pd, g.cuda(), bd, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
        assert pd._version > version
        parts = range(shape[0]) if len(shape) == 4 else [slice(None)]
        for e in parts:
            want_p, want_b = orc.muon_step(p[e].numpy(), g[e].numpy(), buf[e].numpy(), 0.02, 0.9, nesterov, 0.1)
            # the step is 0.02 of a matrix whose norm is above p's: its relative error counts in full
            assert _rel(pd[e], want_p) <= FP32_TOL
            assert _rel(bd[e], want_b) <= 1e-6


def test_muon_optimizer_trains_and_resumes():
    torch.manual_seed(0)
    layer = kan_amd.ChebyKANLayer(12, 9, 4).cuda()
    opt = kan_amd.optim.Muon(layer.parameters(), lr=0.05)
    x = torch.randn(256, 12, device="cuda")
    y = torch.sin(x[:, :9])
    losses = []
    for k in range(30):
        opt.zero_grad()
        loss = ((layer(x) - y) ** 2).mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if k == 15:
            saved = [{n: v.clone() for n, v in layer.state_dict().items()}, opt.state_dict()]
    assert losses[-1] < 0.5 * losses[0]
    other = kan_amd.ChebyKANLayer(12, 9, 4).cuda()
    other.load_state_dict(saved[0])
    opt2 = kan_amd.optim.Muon(other.parameters(), lr=0.05)
    opt2.load_state_dict({"state": {k: {n: t.clone() for n, t in v.items()} for k, v in saved[1]["state"].items()},
                          "param_groups": saved[1]["param_groups"]})
    assert set(opt2.state[other.cheby_coeffs]) == {"momentum_buffer"}


def test_strides_of_dimensions_of_one():
    g = torch.randn(6, 8, 10, device="cuda")
    for v in (g[::6, ::8, ::10], g[:, ::8, :], g[:, :, ::10], g[:1, :, ::10], g[2:3].transpose(1, 2)):
        got = kan_amd.functional.orthogonalize(v)
        assert got.shape == v.shape and torch.equal(got, kan_amd.functional.orthogonalize(v.clone(memory_format=torch.contiguous_format)))
