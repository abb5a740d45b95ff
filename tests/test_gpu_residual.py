"""Norms around a residual block against the 64-bit definition, in every combination of parts.

Bounds: the oracle gives with each result its size, the same expression over absolute values. An fp32
result is a product and sum of at most 24 roundings of such terms, and of row means whose
sums run over at most dim / 256 + 16 terms in sequence (a thread's, then a tree): (48 + dim / 256) 2^-24 of the
size covers both twice. Gradients of parameters add sums over rows: at most rows in sequence. A result in
bf16 adds half a step: of 8 significant bits, 2^-7 apart in [1, 2), so at most 2^-8 of its value; the factor r's relative error enters through the size.
"""
import numpy as np
import pytest
import torch

import kan_amd
from oracle import block_oracle as orc

pytestmark = pytest.mark.gpu
f = kan_amd.functional
F32, BF16 = torch.float32, torch.bfloat16
PARAMS = ("post_weight", "post_bias", "next_weight", "next_bias")


def half_step(t):
    return torch.finfo(t).eps / 2  # 2^-8 and 2^-24


def make(rows, dim, x_dtype, y_dtype, p_dtype, parts, seed):
    """Inputs by name; parts of "y", "post", "next", "bias", "gate", "rows" (a gate a row)."""
    g = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g)

    v = {"x": (2 * randn(rows, dim) + 0.5).to(x_dtype)}
    if "y" in parts:
        v["y"] = (0.4 * randn(rows, dim) - 0.2).to(y_dtype)
    for which in ("post", "next"):
        if which in parts:
            v[which + "_weight"] = (1 + 0.3 * randn(dim)).to(p_dtype)
            if "bias" in parts:
                v[which + "_bias"] = (0.2 * randn(dim)).to(p_dtype)
    if "gate" in parts:
        v["gate"] = (0.5 * randn(dim)).to(p_dtype)
    if "rows" in parts:
        v["gate"] = (0.5 * randn(rows, dim)).to(y_dtype)
    grads = {"out": randn(rows, dim).to(x_dtype), "h": randn(rows, dim).to(y_dtype)}
    return v, grads


def run(v, norm, eps, scale, drop, state, dtype, call=0):
    if "y" not in v:
        return {"h": f.row_norm(v["x"], v["next_weight"], v.get("next_bias"), norm=norm, eps=eps, dtype=dtype)}
    kw = {k: v[k] for k in PARAMS + ("gate",) if k in v}
    got = f.residual_norm(v["x"], v["y"], norm=norm, eps=eps, scale=scale, dropout=drop, dropout_state=state,
                          dropout_call=call, **kw)
    return {"out": got[0], "h": got[1]} if "next_weight" in v else {"out": got}


def compare(name, got, want, size, roundings):
    want, size = torch.from_numpy(np.asarray(want)), torch.from_numpy(np.asarray(size))
    err = (got.detach().cpu().double() - want).abs()
    # the type's own half step, on a value that is off by the arithmetic's error
    limit = roundings * 2.0 ** -24 * size * (1 + half_step(got.dtype)) + half_step(got.dtype) * want.abs() + 1e-37
    worst = (err / limit).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} of its bound at element {int((err / limit).argmax())}"


def check(rows, dim, x_dtype, y_dtype, p_dtype, parts, norm, drop=0.0, seed=1, scale=0.7, eps=1e-5):
    v, grads = make(rows, dim, x_dtype, y_dtype, p_dtype, parts, seed)
    state = torch.tensor([2 ** 40 + seed, 17])
    dev = {k: t.cuda().requires_grad_() for k, t in v.items()}
    got = run(dev, norm, eps, scale, drop, state.cuda(), y_dtype)
    assert got["h" if "y" not in parts else "out"].dtype == (y_dtype if "y" not in parts else x_dtype)
    given = [grads[k].cuda() for k in got]
    dv = torch.autograd.grad(list(got.values()), list(dev.values()), given)
    keep = orc.keep_mask(2 ** 40 + seed, 17, rows, dim, drop) if drop else None
    want = orc.residual(**{k: t.double().numpy() for k, t in v.items()}, norm=norm, eps=eps, scale=scale, keep=keep,
                        p=drop, **{"d" + k: grads[k].double().numpy() for k in got})
    k = 48 + dim / 256
    for name, t in got.items():
        compare(name, t, *want[name], k)
    for name, t in zip(dev, dv):
        assert t.dtype == v[name].dtype and t.shape == v[name].shape
        compare("d" + name, t, *want[name], k + (rows if t.dim() == 1 else 0))
    with torch.no_grad():  # without a graph the same bits
        again = run({k: t.detach() for k, t in dev.items()}, norm, eps, scale, drop, state.cuda(), y_dtype)
    for name in got:
        assert torch.equal(again[name], got[name])


ALL = {"y", "post", "next", "bias", "gate"}


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 9, 63, 64, 65, 130, 257, 500, 512, 777, 1000, 1024, 1029, 2048, 2051, 4100, 8192,
                                 8200, 16384, 20001])
def test_widths(dim, norm):
    check(5, dim, F32, F32, F32, ALL, norm)
    check(3, dim, BF16, BF16, BF16, ALL, norm, drop=0.3, seed=2)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 17, 255, 1025, 3000])
@pytest.mark.parametrize("dim", [10, 96, 300, 520])
def test_rows(rows, dim):
    check(rows, dim, F32, BF16, F32, ALL, "layer", drop=0.1)


@pytest.mark.parametrize("x_dtype", [F32, BF16])
@pytest.mark.parametrize("y_dtype", [F32, BF16])
@pytest.mark.parametrize("p_dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [96, 1001])
def test_types(x_dtype, y_dtype, p_dtype, dim):
    check(9, dim, x_dtype, y_dtype, p_dtype, ALL, "rms")
    check(9, dim, x_dtype, y_dtype, p_dtype, {"y", "post", "next", "rows"}, "layer", drop=0.5)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("parts", [
    {"y"}, {"y", "gate"}, {"y", "rows"}, {"y", "post"}, {"y", "post", "bias"}, {"y", "next"}, {"y", "next", "bias", "rows"},
    {"y", "post", "next"}, {"y", "post", "bias", "rows"}, {"next"}, {"next", "bias"}])
@pytest.mark.parametrize("drop", [0.0, 0.25, 1.0])
def test_parts(parts, norm, drop):
    if "y" not in parts and drop:
        pytest.skip("dropout is the branch's")
    for dim in (48, 700):
        check(6, dim, F32, F32, F32, parts, norm, drop=drop)
        check(6, dim, F32, BF16, F32, parts, norm, drop=drop)


def test_gradients_that_are_not_wanted():
    """Each gradient alone has the bits that it has among all, also where only one output has one."""
    v, grads = make(33, 200, F32, BF16, F32, ALL, 3)
    for drop in (0.0, 0.2):
        for outputs in (("out", "h"), ("out",), ("h",)):
            def grad(names):
                dev = {k: t.cuda().requires_grad_(k in names) for k, t in v.items()}
                got = run(dev, "layer", 1e-5, 1.0, drop, 5, BF16)
                return dict(zip(names, torch.autograd.grad([got[k] for k in outputs], [dev[k] for k in names],
                                                           [grads[k].cuda() for k in outputs], allow_unused=True)))

            every = grad(list(v))
            for name in v:
                alone = grad([name])[name]
                if alone is None:
                    assert every[name] is None or not every[name].any()
                else:
                    assert torch.equal(alone, every[name]), (name, outputs)
    # the gradients where one output has none are those for zeros there
    dev = {k: t.cuda().requires_grad_() for k, t in v.items()}
    got = run(dev, "layer", 1e-5, 1.0, 0.0, None, BF16)
    alone = torch.autograd.grad(got["h"], list(dev.values()), grads["h"].cuda(), retain_graph=True)
    zeros = torch.autograd.grad(list(got.values()), list(dev.values()), [torch.zeros_like(got["out"]), grads["h"].cuda()])
    for a, b in zip(alone, zeros):
        assert torch.equal(a, b)


def test_layouts():
    """Strided, transposed, expanded and unaligned tensors give what their copies give; leading dimensions stay."""
    torch.manual_seed(0)
    rows, dim = 12, 72
    wide = torch.randn(rows, 3 * dim + 5, device="cuda")
    w = torch.rand(dim, 2, device="cuda")[:, 0]
    x, y = wide[:, 1:dim + 1], wide[:, dim + 2:2 * dim + 2].bfloat16()
    cases = [(x, y, w), (x.t().contiguous().t(), y, w), (x, y.t().contiguous().t(), w.expand(dim)),
             (x[:1].expand(rows, dim), y, None), (x, y, x), (x.view(1, rows, dim).expand(2, rows, dim), y.expand(2, rows, dim), w),
             (x.reshape(3, 4, dim), y.reshape(3, 4, dim), w), (x[0], y[0], w), (x[::2], y[::2], y[::2]), (x[:0], y[:0], w)]
    for x, y, gate in cases:
        leaf = [t.detach().clone(memory_format=torch.contiguous_format) if t is not None else None for t in (x, y, gate)]

        def call(x, y, gate):
            args = [None if t is None else t.detach().requires_grad_() for t in (x, y, gate)]
            out, h = f.residual_norm(args[0], args[1], gate=args[2], post_weight=w, next_weight=w, scale=0.5)
            assert out.shape == h.shape == x.shape and out.dtype == x.dtype and h.dtype == y.dtype
            # upstream gradients that are no dense rows
            up = torch.ones(1, device="cuda", dtype=out.dtype).expand(out.shape), torch.ones_like(h).t().contiguous().t() \
                if h.dim() == 2 else torch.ones_like(h)
            return [out, h, *torch.autograd.grad((out, h), [t for t in args if t is not None], up)]

        for a, b in zip(call(x, y, gate), call(*leaf)):
            assert torch.equal(a, b)


def test_large_and_small_values():
    """Rows of zeros, of one value, of huge and of tiny ones."""
    dim = 300
    x = torch.randn(6, dim)
    x[0] = 0
    x[1] = 3.0
    x[2] *= 1e15
    x[3] *= 1e-15
    x[4] = 0
    x[4, 7] = 1e-3
    w = torch.ones(dim)
    for norm in ("rms", "layer"):
        xd = x.cuda().requires_grad_()
        h = f.row_norm(xd, w.cuda(), norm=norm, eps=1e-6)
        dx, = torch.autograd.grad(h, xd, torch.ones_like(h) + torch.arange(dim, device="cuda"))
        want = orc.residual(x.double().numpy(), norm=norm, next_weight=w.double().numpy(),
                            dh=np.ones((6, dim)) + np.arange(dim))
        compare("h", h, *want["h"], 50)
        compare("dx", dx, *want["x"], 50)
    assert torch.isnan(f.row_norm(torch.tensor([[1.0, float("nan")], [1.0, 2.0]], device="cuda"), torch.ones(2, device="cuda"))
                       ).tolist() == [[True, True], [False, False]]


def test_repeats_bit_for_bit_and_changed_inputs_are_refused():
    v, grads = make(700, 333, BF16, BF16, F32, ALL, 4)

    def once():
        dev = {k: t.cuda().requires_grad_() for k, t in v.items()}
        got = run(dev, "rms", 1e-6, 1.0, 0.1, 9, BF16)
        return dev, got, torch.autograd.grad(list(got.values()), list(dev.values()), [grads[k].cuda() for k in got],
                                             retain_graph=True)

    (dev, got, a), (_, _, b) = once(), once()
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    with torch.no_grad():
        dev["x"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(got["h"], dev["x"], torch.ones_like(got["h"]))
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    h = f.row_norm(x, torch.ones(8, device="cuda"))
    g, = torch.autograd.grad(h.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(h.sum(), x, create_graph=True)


def test_refusals_on_the_device():
    x, w = torch.zeros(2, 4, device="cuda"), torch.ones(4, device="cuda")
    for call, error in ((lambda: f.row_norm(x, w[:3]), "weight"), (lambda: f.row_norm(x, torch.ones(4)), "cpu"),
                        (lambda: f.row_norm(x.double(), w), "float32 or bfloat16"),
                        (lambda: f.row_norm(x, w, dtype=torch.float16), "float32 or bfloat16"),
                        (lambda: f.residual_norm(x, x[:1]), "shape"), (lambda: f.residual_norm(x, x, gate=w[:2]), "gate"),
                        (lambda: f.residual_norm(x, x, post_bias=w), "weight"),
                        (lambda: f.residual_norm(x, x, next_bias=w), "weight"),
                        (lambda: f.residual_norm(x, x, dropout=0.5, dropout_state=torch.zeros(2, device="cuda")), "state")):
        with pytest.raises(RuntimeError, match=error):
            call()
    with pytest.raises(ValueError, match="state"):
        f.residual_norm(x, x, dropout=0.5)
    with pytest.raises(ValueError, match="probability"):
        f.residual_norm(x, x, dropout=-0.5, dropout_state=1)
