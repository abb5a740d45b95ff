"""Few-row mixtures whose rows crowd on few experts: an expert's slots fill several blocks' shares, up to and past their ends.

Bounds as the other tests of the few-row form: weights 1e-6, y 5e-6 of its norm against the 64-bit sum."""
import numpy as np
import pytest
import torch

import kan_amd
from kan_amd import _lib
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
F32, BF16 = torch.float32, torch.bfloat16


def check(counts, rest, top_k, experts, in_dim, out_dim, degree, c_dtype):
    """Rows whose first choice is expert e for counts[e] of them, the others by chance; ``rest``: rows with no expert."""
    rows = sum(counts.values()) + rest
    g = torch.Generator().manual_seed(rows + degree)
    # an input of its own for every expert says how much the row wants it
    x = torch.randn(rows, in_dim + experts, generator=g)
    wants = 0.5 * torch.randn(rows, experts, generator=g)
    first = torch.tensor([e for e, n in counts.items() for _ in range(n)])[torch.randperm(rows - rest, generator=g)]
    wants[torch.arange(rows - rest), first] = 4.0
    x[:, in_dim:] = wants
    x[rows - rest:] = float("nan")  # no logit is a number there: no expert
    gate = torch.zeros(experts, in_dim + experts)
    gate[:, in_dim:] = torch.eye(experts)
    coeffs = (torch.randn(experts, in_dim + experts, out_dim, degree + 1, generator=g) / (in_dim * (degree + 1))).to(c_dtype)
    desc = _lib.CkanMixtureDesc(rows, experts, top_k, in_dim + experts, out_dim, degree, 0, 1, 1, 1, 0, 0, 0, 1.0)
    assert _lib.load().ckan_mixture_few(desc) == 1
    with torch.no_grad():
        y, w, idx = (t.cpu() for t in f.kan_mixture(x.cuda(), gate.cuda(), coeffs.cuda(), top_k))
    full = rows - rest
    want_w, want_idx = orc.route(wants[:full].double().numpy(), top_k)
    assert np.array_equal(idx[:full].numpy(), want_idx) and np.array_equal(want_idx[:, 0], first.numpy())
    assert np.abs(w[:full].numpy() - want_w).max() <= 1e-6
    want = orc.kan_experts(x[:full].double().numpy(), coeffs.double().numpy(), want_idx, want_w)
    assert np.linalg.norm(y[:full].double().numpy() - want) <= 5e-6 * np.linalg.norm(want)
    # row by row too, a slot left out would hardly show in the norm of all: no row has less than a tenth of the mean row's norm
    worst = (np.linalg.norm(y[:full].double().numpy() - want, axis=1) / np.linalg.norm(want, axis=1)).max()
    assert worst <= 5e-5
    assert (idx[full:] == -1).all() and not w[full:].any() and not y[full:].any()


@pytest.mark.parametrize("c_dtype", [F32, BF16])
@pytest.mark.parametrize("counts", [
    {0: 64, 3: 1}, {3: 65}, {0: 128}, {1: 129}, {2: 63, 3: 65}, {0: 97, 1: 96, 2: 31, 3: 31}, {3: 200}, {0: 130, 1: 2, 3: 66}],
    ids=str)
def test_shares_of_an_expert(counts, c_dtype):
    check(counts, 0, 1, 4, 20, 66, 4, c_dtype)


@pytest.mark.parametrize("c_dtype", [F32, BF16])
@pytest.mark.parametrize("counts,rest,top_k,experts,in_dim,out_dim,degree", [
    ({5: 500}, 0, 2, 16, 50, 70, 3), ({511: 300, 0: 30, 256: 80}, 0, 2, 512, 9, 33, 2), ({63: 250, 62: 6}, 0, 4, 64, 130, 64, 9),
    ({7: 90, 8: 70}, 40, 3, 12, 30, 31, 16), ({1: 400}, 112, 2, 20, 24, 20, 8), ({i: 65 for i in range(0, 15, 2)}, 0, 1, 16, 24, 20, 5)],
    ids=str)
def test_rows_that_crowd(counts, rest, top_k, experts, in_dim, out_dim, degree, c_dtype):
    check(counts, rest, top_k, experts, in_dim, out_dim, degree, c_dtype)


def test_a_row_does_not_depend_on_the_crowd():
    """The same bits for a row among 500 on two experts and among 100 spread over all."""
    torch.manual_seed(1)
    x = torch.randn(500, 48, device="cuda")
    gate, coeffs = torch.randn(16, 48, device="cuda"), torch.randn(16, 48, 40, 6, device="cuda")
    bias = torch.zeros(16, device="cuda")
    bias[[3, 9]] = 5.0
    with torch.no_grad():
        every = f.kan_mixture(x, gate, coeffs, 2, bias=bias)
        some = f.kan_mixture(x[40:140], gate, coeffs, 2, bias=bias)
    for a, b in zip(every, some):
        assert torch.equal(a[40:140], b)
