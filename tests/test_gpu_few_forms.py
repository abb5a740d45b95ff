"""Few-row mixtures on either side of the rules between the forms of the gate and of the products.

Bounds as the other tests of the few-row form: weights 1e-6, y 5e-6 of its norm against the 64-bit sum, and half a step more of
each value of a y in bf16."""
import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
F32, BF16 = torch.float32, torch.bfloat16


def check(rows, in_dim, out_dim, degree, experts, top_k, x_dtype=F32, g_dtype=F32, c_dtype=F32, few=1, bias=None, **how):
    g = torch.Generator().manual_seed(rows + experts)
    x = torch.randn(rows, in_dim, generator=g).to(x_dtype)
    gate = (2 * torch.randn(experts, in_dim, generator=g) / in_dim ** 0.5).to(g_dtype)
    coeffs = (torch.randn(experts, in_dim, out_dim, degree + 1, generator=g) / (in_dim * (degree + 1))).to(c_dtype)
    code = {F32: 0, BF16: 1}
    desc = _lib.CkanMixtureDesc(rows, experts, top_k, in_dim, out_dim, degree, 0, 1, 1, 1, code[x_dtype], code[g_dtype],
                                code[c_dtype], 1.0)
    assert _lib.load().ckan_mixture_few(desc) == few
    with torch.no_grad():
        y, w, idx = (t.cpu() for t in f.kan_mixture(x.cuda(), gate.cuda(), coeffs.cuda(), top_k, **how,
                                                          bias=None if bias is None else bias.cuda()))
    if few:
        logits = (x.double() @ gate.double().t()).float()
        want_w, want_idx = orc.route(logits.double().numpy(), top_k, bias=None if bias is None else bias.numpy(), **how)
        assert np.array_equal(idx.numpy(), want_idx)
        assert np.abs(w.numpy() - want_w).max() <= 1e-6
    want = orc.kan_experts(x.double().numpy(), coeffs.double().numpy(), idx.numpy(), w.double().numpy())
    err = np.abs(y.double().numpy() - want)
    if x_dtype == BF16:
        err = np.maximum(err - 2.0 ** -8 * np.abs(want), 0)
    assert np.linalg.norm(err) <= 5e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("rows", [1, 2, 9, 70])
@pytest.mark.parametrize("experts,in_dim", [(127, 40), (128, 40), (128, 7), (129, 65), (300, 12), (512, 24), (64, 1024), (64, 1025)])
def test_gates_of_many_experts(rows, experts, in_dim):
    for x_dtype, g_dtype in ((F32, F32), (BF16, F32), (BF16, BF16)):
        check(rows, in_dim, 18, 2, experts, 3, x_dtype, g_dtype)


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("experts,groups,top_groups", [(128, 8, 3), (192, 64, 20), (512, 4, 2), (130, 2, 1)])
def test_groups_of_many_experts(rows, experts, groups, top_groups):
    bias = 0.171 * torch.randint(-3, 4, (experts,), generator=torch.Generator().manual_seed(2)).float()
    check(rows, 33, 20, 3, experts, 4, bias=bias, score="sigmoid", groups=groups, top_groups=top_groups)
    check(rows, 33, 20, 3, experts, 4, groups=groups, top_groups=top_groups, renormalize=False, scale=1.5)


@pytest.mark.parametrize("c_dtype", [F32, BF16])
@pytest.mark.parametrize("case", [
    (4, 30, 34, 5, 40, 16), (5, 30, 34, 5, 40, 16), (8, 30, 33, 3, 64, 8), (8, 30, 33, 3, 64, 9), (2, 20, 70, 9, 64, 33),
    (8, 17, 16, 16, 100, 64), (5, 640, 700, 2, 14, 13), (5, 640, 700, 5, 14, 13)], ids=lambda c: "-".join(map(str, c)))
def test_few_rows_of_many_slots(case, c_dtype):
    """64 slots and more of up to 8 rows, in experts of few and of many coefficients."""
    for x_dtype in (F32, BF16):
        check(*case, x_dtype, F32, c_dtype)


@pytest.mark.parametrize("rows,experts,top_k,in_dim,crowd", [(300, 16, 2, 40, True), (300, 16, 2, 40, False), (5, 300, 16, 30, False),
                                                            (1, 200, 3, 50, False), (70, 512, 4, 20, True)])
def test_replays_of_a_captured_call(rows, experts, top_k, in_dim, crowd):
    """New rows and another crowd at every replay, with eager calls between."""
    torch.manual_seed(rows)
    gate, coeffs = torch.randn(experts, in_dim, device="cuda"), torch.randn(experts, in_dim, 24, 5, device="cuda")
    x, bias = torch.zeros(rows, in_dim, device="cuda"), torch.zeros(experts, device="cuda")
    with torch.no_grad():
        f.kan_mixture(x, gate, coeffs, top_k, bias=bias)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = f.kan_mixture(x, gate, coeffs, top_k, bias=bias)
        for i in range(5):
            x.normal_()
            bias.zero_()
            if crowd:
                bias[3 * i:3 * i + top_k] = 5.0
            graph.replay()
            want = f.kan_mixture(x.clone(), gate, coeffs, top_k, bias=bias.clone())
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
