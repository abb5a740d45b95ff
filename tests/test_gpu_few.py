"""A whole mixture layer for few rows against the 64-bit definition.

Bounds: the logits are rounded once (2^-24), which a score carries as |l| 2^-24 or so and a weight under
1e-6 of the largest, as ``route``'s own. y in fp32: a basis value by the recurrence is off by at most about degree^2 / 2 half
steps of 1 (each of its steps adds one, and errors grow linearly in the degree), tanh by 2 more; the sums run
over in * degree / 256 terms in sequence and a tree: the norm-wise 5e-6 of the experts' fp32 forward. y in bf16 adds its half step,
2^-8 of each value.
"""
import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
F32, BF16 = torch.float32, torch.bfloat16


def make(rows, in_dim, out_dim, degree, experts, x_dtype, g_dtype, c_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, in_dim, generator=g).to(x_dtype)
    gate = (2 * torch.randn(experts, in_dim, generator=g) / in_dim ** 0.5).to(g_dtype)
    coeffs = (torch.randn(experts, in_dim, out_dim, degree + 1, generator=g) / (in_dim * (degree + 1))).to(c_dtype)
    return x, gate, coeffs


def check(x, gate, coeffs, top_k, **how):
    logits = (x.double() @ gate.double().t()).float()
    kw = {k: (v.numpy() if isinstance(v, torch.Tensor) else v) for k, v in how.items()}
    w, idx = orc.route(logits.double().numpy(), top_k, **kw)
    want = orc.kan_experts(x.double().numpy(), coeffs.double().numpy(), idx, w)
    dev = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in how.items()}
    with torch.no_grad():
        y, gw, gi = f.kan_mixture(x.cuda(), gate.cuda(), coeffs.cuda(), top_k, **dev)
    assert y.dtype == x.dtype and gw.dtype == F32 and gi.dtype == torch.int64
    assert np.array_equal(gi.cpu().numpy(), idx)
    assert np.abs(gw.cpu().numpy() - w).max() <= 1e-6 * max(1.0, np.abs(w).max())
    err = np.abs(y.double().cpu().numpy() - want)
    if x.dtype == BF16:
        err = np.maximum(err - 2.0 ** -8 * np.abs(want), 0)
    assert np.linalg.norm(err) <= 5e-6 * np.linalg.norm(want) + 1e-30
    return y, gw, gi


CASES = [
    # rows, in, out, degree, experts, top_k, score, groups, top_groups, bias
    (1, 1, 1, 1, 1, 1, "softmax", 1, 1, False),
    (1, 64, 64, 8, 8, 2, "softmax", 1, 1, False),
    (1, 300, 257, 5, 8, 2, "softmax", 1, 1, True),
    (1, 2048, 130, 8, 4, 2, "sigmoid", 1, 1, False),
    (2, 33, 65, 16, 5, 5, "sigmoid", 1, 1, True),
    (3, 129, 7, 3, 64, 4, "sigmoid", 8, 4, True),
    (7, 500, 300, 5, 6, 2, "softmax", 1, 1, False),
    (8, 65, 1000, 2, 16, 1, "softmax", 4, 1, False),
    (9, 16, 16, 13, 512, 8, "softmax", 1, 1, False),
    (17, 100, 63, 4, 3, 2, "softmax", 1, 1, False),
    (40, 96, 48, 7, 12, 3, "sigmoid", 3, 2, True),
    (64, 31, 200, 1, 64, 4, "softmax", 1, 1, False),
    (256, 24, 40, 6, 64, 4, "softmax", 1, 1, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("x_dtype,g_dtype,c_dtype", [(F32, F32, F32), (F32, F32, BF16), (BF16, F32, BF16), (BF16, BF16, F32)])
def test_against_definition(case, x_dtype, g_dtype, c_dtype):
    rows, in_dim, out_dim, degree, experts, top_k, score, groups, top_groups, biased = case
    x, gate, coeffs = make(rows, in_dim, out_dim, degree, experts, x_dtype, g_dtype, c_dtype, rows + degree)
    desc = _lib.CkanMixtureDesc(rows, experts, top_k, in_dim, out_dim, degree, 0, 1, 1, 1, 0, 0, 0, 1.0)
    assert _lib.load().ckan_mixture_few(desc) == 1
    bias = 0.171 * torch.randint(-3, 4, (experts,), generator=torch.Generator().manual_seed(1)).float() if biased else None
    check(x, gate, coeffs, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups)
    check(x, gate, coeffs, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalize=False, scale=1.5)


@pytest.mark.parametrize("degree", range(1, 17))
def test_degrees(degree):
    for rows, c_dtype in ((1, F32), (1, BF16), (5, F32), (21, BF16)):
        x, gate, coeffs = make(rows, 70, 37, degree, 6, F32, F32, c_dtype, degree)
        x[0] *= 10  # saturated
        check(x, gate, coeffs, 2)


def test_rows_on_one_expert_and_ties():
    """Every row to the same experts (more than a pass serves), equal logits to the lowest index, no expert left."""
    x, gate, coeffs = make(30, 40, 50, 4, 8, F32, F32, F32, 3)
    gate[:] = gate[0]
    _, _, idx = check(x, gate, coeffs, 2)
    assert (idx.cpu() == torch.tensor([0, 1])).all()
    x, gate, coeffs = make(4, 40, 50, 4, 8, F32, F32, F32, 4)
    bias = torch.full((8,), -float("inf"))
    y, w, idx = check(x, gate, coeffs, 2, bias=bias)
    assert (idx == -1).all() and (w == 0).all() and (y == 0).all()
    bias[3] = 0.0
    _, w, idx = check(x, gate, coeffs, 2, bias=bias)
    assert (idx.cpu() == torch.tensor([3, -1])).all()


def test_wide_layers():
    for rows, in_dim, out_dim, c_dtype in ((1, 5000, 300, BF16), (1, 40, 9000, F32), (3, 2048, 2048, BF16), (1, 2049, 2047, F32)):
        x, gate, coeffs = make(rows, in_dim, out_dim, 2, 4, F32, F32, c_dtype, in_dim)
        check(x, gate, coeffs, 2)


@pytest.mark.parametrize("degree", [1, 4, 7, 8, 9, 16])
@pytest.mark.parametrize("c_dtype", [F32, BF16])
def test_many_rows_an_expert(degree, c_dtype):
    """Several passes over the rows of one expert, with 1 to 32 in the last; odd and even outputs, inputs past a chunk's end."""
    for rows, in_dim, out_dim, lean in ((33, 130, 66, 0.0), (48, 37, 65, 0.0), (125, 64, 30, 4.0), (126, 259, 200, 0.5)):
        x, gate, coeffs = make(rows, in_dim, out_dim, degree, 2, F32, F32, c_dtype, rows)
        check(x, gate, coeffs, 1, bias=torch.tensor([0.1 * lean, 0.0]))


def test_an_infinite_coefficient_stays_in_its_output():
    for rows, c_dtype in ((1, F32), (5, BF16), (40, F32), (40, BF16)):
        x, gate, coeffs = (t.cuda() for t in make(rows, 70, 34, 5, 4, F32, F32, c_dtype, 8))
        with torch.no_grad():
            want, _, idx = f.kan_mixture(x, gate, coeffs, 2)
            coeffs[2, 11, 7, 3] = float("inf")
            coeffs[2, 69, 33, 0] = float("nan")
            got, _, again = f.kan_mixture(x, gate, coeffs, 2)
        hit = torch.zeros_like(want, dtype=torch.bool)
        hit[(idx == 2).any(1)[:, None] & torch.isin(torch.arange(34, device="cuda"), torch.tensor([7, 33], device="cuda"))] = True
        assert torch.equal(idx, again) and torch.equal(got[~hit], want[~hit]) and not torch.isfinite(got[hit]).any()


@pytest.mark.parametrize("rows", [1, 2, 20])
def test_large_gates(rows):
    """Gates of more than 2^16 entries, whose logits a launch of their own makes."""
    for in_dim, experts, dtype in ((1100, 64, F32), (130, 512, BF16), (3001, 24, F32)):
        x, gate, coeffs = make(rows, in_dim, 20, 3, experts, F32, dtype, F32, in_dim)
        assert in_dim * experts > 1 << 16
        check(x, gate, coeffs, 3)


def test_many_rows_and_gradients_take_the_parts():
    x, gate, coeffs = (t.cuda() for t in make(300, 40, 30, 4, 4, F32, F32, F32, 6))
    with torch.no_grad():
        y, w, idx = f.kan_mixture(x, gate, coeffs, 2)
        rw, ri = f.route(x @ gate.t(), 2)
        assert torch.equal(w, rw) and torch.equal(idx, ri) and torch.equal(y, f.kan_experts(x, coeffs, ri, rw))
    leaves = [t[:3].clone().requires_grad_() if t is x else t.clone().requires_grad_() for t in (x, gate, coeffs)]
    y, w, idx = f.kan_mixture(*leaves, 2)
    g = torch.autograd.grad(y.square().sum(), leaves)
    assert all(torch.isfinite(t).all() and t.abs().sum() > 0 for t in g)
    with torch.no_grad():
        z, _, _ = f.kan_mixture(*leaves, 2)
    assert ((y - z).norm() / z.norm()).item() <= 1e-5
    none = f.kan_mixture(x[:0], gate, coeffs, 2)
    assert none[0].shape == (0, 30) and none[1].shape == none[2].shape == (0, 2)


def test_layouts():
    x, gate, coeffs = (t.cuda() for t in make(5, 48, 20, 3, 6, F32, F32, F32, 9))
    with torch.no_grad():
        want = f.kan_mixture(x, gate, coeffs, 2)
        for a, b, c in ((x.t().contiguous().t(), gate, coeffs), (torch.cat([x, x], 1)[:, :48], gate.t().contiguous().t(), coeffs),
                        (x, torch.cat([gate.reshape(-1)[:1], gate.reshape(-1)])[1:].view(6, 48), coeffs.transpose(1, 2).contiguous().transpose(1, 2))):
            for u, v in zip(f.kan_mixture(a, b, c, 2), want):
                assert torch.equal(u, v)


@pytest.mark.parametrize("compute", ["fp32", "bf16"])
def test_the_layer_takes_it(compute):
    torch.manual_seed(5)
    layer = kan_amd.MixtureKANLayer(60, 50, 6, experts=8, top_k=2, score="sigmoid", balance=True, compute=compute).cuda()
    x = torch.randn(3, 60, device="cuda")
    with torch.no_grad():
        y = layer(x)
        want, _, idx = f.kan_mixture(x, layer.gate, layer.cheby_coeffs, 2, score="sigmoid", bias=layer.balance_bias)
    assert torch.equal(y, want) and torch.equal(layer._last_indices, idx)
    z = layer(x)
    assert z.requires_grad and ((z - y).norm() / y.norm()).item() <= (1e-5 if compute == "fp32" else 2e-2)
    layer.update_balance()


def test_refusals_on_the_device():
    x, gate, coeffs = (t.cuda() for t in make(2, 8, 6, 3, 4, F32, F32, F32, 1))
    for args, match in (((x[:, :7], gate, coeffs, 2), "x must be"), ((x, gate[:3], coeffs, 2), "gate must be"),
                        ((x, gate, coeffs[0], 2), "coeffs must be"), ((x.double(), gate, coeffs, 2), "float32 or bfloat16"),
                        ((x, gate, coeffs, 5), "top_k"), ((x, gate.cpu(), coeffs, 2), "ROCm device")):
        with pytest.raises(RuntimeError, match=match):
            f.kan_mixture(*args)
    with pytest.raises(RuntimeError, match="bias must be"):
        f.kan_mixture(x, gate, coeffs, 2, bias=torch.zeros(3, device="cuda"))
