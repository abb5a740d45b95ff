"""The products of ChebyKAN experts against the definition in 64 bits.

Bounds on the 2-norm of the error over the 2-norm of the result.  fp32: operands of
22 bits (2^-23 each, rounded), sums of K terms in fp32 and a basis recurrence of up
to 16 steps on a tanh of 2 ulp: a term's error is below 2^-20 (the recurrence takes
an error of t times d^2 at worst near |t| = 1, d on average), 5e-6 with the sums' own.
bf16: basis and gradients carry 11 bits (2^-12), the result one rounding to 8 bits:
at most 2^-8 of each value; 5e-3.  Values that cancel within an expert's sum or
between the slots of a row count against the result's norm, not their own.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import mixture_oracle as orc

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 5e-6, torch.bfloat16: 5e-3}
NAMES = ("y", "dx", "dcoeffs", "dweights")


def _inputs(rows, in_dim, out, degree, experts, top_k, dtype, seed=0, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, in_dim, generator=g).to(dtype)
    c = (torch.randn(experts, in_dim, out, degree + 1, generator=g) / (in_dim * (degree + 1))).to(dtype)
    scores = torch.randn(rows, experts, generator=g) + torch.randn(1, experts, generator=g)
    best, idx = torch.topk(scores, min(top_k, experts), dim=1)
    w = torch.softmax(best, 1).to(wdtype or dtype)
    dy = torch.randn(rows, out, generator=g).to(dtype)
    return x, c, idx, w, dy


def _run(x, c, idx, w, dy):
    xd, cd, wd = (v.cuda().requires_grad_() for v in (x, c, w))
    y = kan_amd.functional.kan_experts(xd, cd, idx.cuda(), wd)
    grads = torch.autograd.grad(y, (xd, cd, wd), dy.cuda())
    return (y.detach(),) + grads


def _check(got, want, dtypes, computed):
    """Each output against the bound of its own type and of the type it was computed in, the larger."""
    for name, a, b, dt in zip(NAMES, got, want, dtypes):
        assert a.dtype == dt, name
        a = a.double().cpu().numpy()
        assert np.isfinite(a).all(), name
        assert np.linalg.norm(a - b) <= max(TOL[dt], TOL[computed]) * np.linalg.norm(b) + 1e-30, name


def _compare(rows, in_dim, out, degree, experts, top_k, dtype, seed=0, edit=None, wdtype=None):
    x, c, idx, w, dy = _inputs(rows, in_dim, out, degree, experts, top_k, dtype, seed, wdtype)
    if edit:
        x, c, idx, w, dy = edit(x, c, idx, w, dy)
    got = _run(x, c, idx, w, dy)
    want = orc.kan_experts(*(v.double().numpy() for v in (x, c)), idx.numpy(), w.double().numpy(),
                           dy.double().numpy())
    _check(got, want, (dtype, dtype, dtype, w.dtype), dtype)
    with torch.no_grad():  # the form without a backward
        y = kan_amd.functional.kan_experts(x.cuda(), c.cuda(), idx.cuda(), w.cuda())
    _check((y,), want[:1], (dtype,), dtype)
    return got, want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,in_dim,out,degree,experts,top_k", [
    (1, 1, 1, 1, 1, 1),
    (1, 64, 48, 8, 4, 2),
    (3, 33, 130, 2, 5, 5),
    (40, 20, 257, 3, 7, 2),
    (129, 31, 20, 4, 3, 1),
    (130, 50, 70, 5, 6, 2),
    (200, 65, 33, 8, 16, 4),
    (257, 16, 40, 9, 2, 2),
    (300, 40, 24, 16, 3, 2),
    (64, 7, 300, 12, 9, 3),
    (1100, 10, 12, 6, 40, 3),
])
def test_against_definition(rows, in_dim, out, degree, experts, top_k, dtype):
    _compare(rows, in_dim, out, degree, experts, top_k, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropped_and_repeated_slots(dtype):
    def edit(x, c, idx, w, dy):
        idx = idx.clone()
        idx[0] = -1                    # a row with no expert
        idx[5, 0], idx[6, 1] = -1, 99  # single slots without one, either side of the range
        idx[7] = 2                     # one expert twice
        idx[idx == 3] = 1              # an expert without rows
        return x, c, idx, w, dy

    (y, dx, dc, dw), _ = _compare(150, 24, 40, 6, 5, 2, dtype, edit=edit)
    assert (y[0] == 0).all() and (dx[0] == 0).all() and (dw[0] == 0).all()
    assert (dc[3] == 0).all() and dw[5, 0] == 0 and dw[6, 1] == 0


def test_all_slots_dropped_and_one_expert_for_all():
    _compare(70, 12, 9, 3, 4, 2, torch.float32, edit=lambda x, c, i, w, dy: (x, c, i * 0 - 1, w, dy))
    _compare(700, 12, 9, 3, 4, 2, torch.float32, edit=lambda x, c, i, w, dy: (x, c, i * 0 + 3, w, dy))


def test_weights_of_another_type():
    _compare(90, 20, 30, 4, 4, 2, torch.bfloat16, wdtype=torch.float32)
    _compare(90, 20, 30, 4, 4, 2, torch.float32, wdtype=torch.bfloat16)


def test_scales_of_coefficients_and_gradients():
    """Powers of two that differ by expert, far beyond fp16's range."""
    def edit(x, c, idx, w, dy):
        c = c * torch.tensor([2.0 ** -60, 1.0, 2.0 ** 40, 2.0 ** -20]).view(-1, 1, 1, 1)
        return x, c, idx, w, dy * 2.0 ** -50

    x, c, idx, w, dy = edit(*_inputs(120, 16, 24, 5, 4, 1, torch.float32, 3))
    got = _run(x, c, idx, w, dy)
    want = orc.kan_experts(x.numpy(), c.numpy(), idx.numpy(), w.numpy(), dy.numpy())
    for e in range(4):  # each expert's rows and gradients on their own
        r = (idx[:, 0] == e).numpy()
        for k, rows in ((0, r), (1, r), (3, r), (2, e)):
            a, b = got[k].double().cpu().numpy()[rows], want[k][rows]
            assert np.linalg.norm(a - b) <= TOL[torch.float32] * np.linalg.norm(b), (NAMES[k], e)


def test_saturated_inputs_and_nan_stay_in_their_rows():
    x, c, idx, w, dy = _inputs(140, 18, 20, 7, 3, 2, torch.float32, 4)
    x[2] = 30.0   # tanh is 1 in fp32: the derivative is 0, not NaN
    x[3] = -float("inf")
    clean = _run(x, c, idx, w, dy)
    for v in clean:
        assert torch.isfinite(v).all()
    assert (clean[1][2] == 0).all()
    x[4, 5] = float("nan")
    got = _run(x, c, idx, w, dy)
    rest = torch.arange(140) != 4
    assert torch.isnan(got[0][4]).all()
    for k in (0, 1, 3):
        assert torch.equal(got[k][rest], clean[k][rest]), NAMES[k]
    hit = set(idx[4].tolist())
    for e in range(3):
        if e not in hit:
            assert torch.equal(got[2][e], clean[2][e])
        else:  # only the poisoned input's coefficients
            assert torch.isnan(got[2][e, 5, :, 1:]).all()
            keep = torch.arange(18) != 5
            assert torch.equal(got[2][e][keep], clean[2][e][keep])


def test_infinite_coefficient_stays_in_its_expert_and_output():
    x, c, idx, w, dy = _inputs(60, 10, 14, 4, 3, 1, torch.float32, 5)
    clean = _run(x, c, idx, w, dy)[0]
    c[1, 2, 3, 2] = float("inf")
    got = _run(x, c, idx, w, dy)[0]
    mine = (idx[:, 0] == 1)
    assert not torch.isfinite(got[mine.cuda(), 3]).any()
    got[mine.cuda(), 3] = clean[mine.cuda(), 3]
    assert torch.equal(got, clean)


def test_gradient_against_differences():
    x, c, idx, w, dy = _inputs(6, 5, 4, 3, 3, 2, torch.float32, 6)
    got = [v.double().cpu().numpy() for v in _run(x, c, idx, w, dy)[1:]]
    args = [v.double().numpy() for v in (x, c, w)]
    rng = np.random.RandomState(1)
    for k in range(3):
        u = rng.randn(*args[k].shape)
        h = 1e-5

        def f(s):
            v = [a.copy() for a in args]
            v[k] += s * h * u
            return (orc.kan_experts(v[0], v[1], idx.numpy(), v[2]) * dy.numpy()).sum()

        want = (f(1) - f(-1)) / (2 * h)
        # the difference's own error is h^2 of a third derivative of size about the first
        assert abs((got[k] * u).sum() - want) <= 1e-5 * (np.linalg.norm(got[k]) * np.linalg.norm(u))


def test_layouts_streams_partial_gradients_and_repeats():
    x, c, idx, w, dy = _inputs(150, 24, 40, 6, 5, 2, torch.float32, 7)
    base = _run(x, c, idx, w, dy)
    again = _run(x, c, idx, w, dy)
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    # strided inputs
    xs = torch.zeros(150, 60)
    xs[:, 10:34] = x
    y = kan_amd.functional.kan_experts(xs.cuda()[:, 10:34], c.permute(3, 0, 1, 2).contiguous().cuda().permute(1, 2, 3, 0),
                                       idx.t().contiguous().cuda().t(), w.t().contiguous().cuda().t())
    assert torch.equal(y, base[0])
    # contiguous tensors at addresses that no vector load can take
    off = torch.zeros(150 * 24 + 1)
    off[1:] = x.reshape(-1)
    offc = torch.zeros(c.numel() + 1)
    offc[1:] = c.reshape(-1)
    y = kan_amd.functional.kan_experts(off.cuda()[1:].view(150, 24), offc.cuda()[1:].view(c.shape), idx.cuda(), w.cuda())
    assert torch.equal(y, base[0])
    # another stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _run(x, c, idx, w, dy)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, other))
    # one gradient at a time gives the same bits
    for k in range(3):
        t = [v.cuda() for v in (x, c, w)]
        t[k].requires_grad_()
        y = kan_amd.functional.kan_experts(t[0], t[1], idx.cuda(), t[2])
        g, = torch.autograd.grad(y, (t[k],), dy.cuda())
        assert torch.equal(g, base[k + 1]), NAMES[k + 1]
    # no rows
    e = torch.empty(0, 24, device="cuda", requires_grad=True)
    cd = c.cuda().requires_grad_()
    y = kan_amd.functional.kan_experts(e, cd, torch.empty(0, 2, dtype=torch.int64, device="cuda"),
                                       torch.empty(0, 2, device="cuda"))
    assert y.shape == (0, 40)
    y.sum().backward()
    assert (cd.grad == 0).all() and e.grad.shape == (0, 24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("degree", [1, 2, 3, 5, 7, 8, 10, 11, 13, 14, 15, 16])
def test_few_slots(degree, dtype):
    """The streaming forward: odd output counts put bf16 rows on odd halves of a dword."""
    def edit(x, c, idx, w, dy):
        idx = idx.clone()
        idx[0] = -1
        idx[1:20, 0] = 1  # more rows of one expert than a pass over its coefficients serves
        return x, c, idx, w, dy

    _compare(21, 67, 77, degree, 3, 2, dtype, seed=degree, edit=edit)


def test_streaming_and_tile_forwards_agree():
    """The same rows through calls of few slots and one of many."""
    x, c, idx, w, _ = (v.cuda() for v in _inputs(700, 130, 200, 8, 4, 2, torch.float32, 11))
    whole = kan_amd.functional.kan_experts(x, c, idx, w)
    parts = torch.cat([kan_amd.functional.kan_experts(x[r:r + 7], c, idx[r:r + 7], w[r:r + 7]) for r in range(0, 700, 7)])
    assert ((whole - parts).norm() / whole.norm()).item() <= 2 * TOL[torch.float32]


def test_one_expert_is_the_layer():
    """A mixture of one expert of weight 1 is the framework's own layer."""
    torch.manual_seed(1)
    layer = kan_amd.ChebyKANLayer(48, 36, 8).cuda()
    x = torch.randn(200, 48, device="cuda")
    y = kan_amd.functional.kan_experts(x, layer.cheby_coeffs.detach()[None], torch.zeros(200, 1, dtype=torch.int64, device="cuda"),
                                       torch.ones(200, 1, device="cuda"))
    want = layer(x)
    assert ((y - want).norm() / want.norm()).item() <= 2 * TOL[torch.float32]


def test_second_derivative_is_refused():
    x = torch.randn(5, 6, device="cuda", requires_grad=True)
    c = torch.randn(3, 6, 4, 3, device="cuda")
    idx = torch.tensor([[0, 2]] * 5, device="cuda")
    y = kan_amd.functional.kan_experts(x, c, idx, torch.ones(5, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)
