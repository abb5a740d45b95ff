"""The residual stack, its loss and its serving form together, as a network runs them."""
import os
import sys

import pytest
import torch

import kan_amd
from oracle import block_oracle as orc
from oracle import chebykan_oracle  # noqa: F401  (the layers' oracle, by its closed form below)

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
f = kan_amd.functional


def layer64(x, coeffs):
    """A ChebyKAN layer by the closed form in 64 bits."""
    n = torch.arange(coeffs.shape[2], dtype=torch.float64)
    phi = torch.cos(n * torch.acos(torch.tanh(x))[..., None])
    return torch.tensordot(phi, coeffs.permute(0, 2, 1).contiguous(), dims=2)


def norm64(x, w, b, norm, eps):
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    return x if b is None else x + b


def stack64(model, p, x, keeps):
    """ResidualKAN of ChebyKAN layers from parameters p (by name), in 64 bits."""
    def at(name, i):
        return p.get(f"{name}.{i}")

    h = norm64(x, at("pre_weight", 0), at("pre_bias", 0), model.norm, model.eps)
    for i in range(len(model.layers)):
        u = layer64(h, p[f"layers.{i}.cheby_coeffs"])
        if at("post_weight", i) is not None:
            u = norm64(u, at("post_weight", i), at("post_bias", i), model.norm, model.eps)
        if keeps is not None:
            u = u * keeps[i] / (1 - model.dropout)
        g = at("gate", i)
        x = x + model.scale * (1.0 if g is None else g) * u
        w = at("pre_weight", i + 1)
        h = x if w is None else norm64(x, w, at("pre_bias", i + 1), model.norm, model.eps)
    return h


@pytest.mark.parametrize("norm,post,gate,drop,final", [("rms", True, 0.3, 0.0, True), ("layer", True, 0.3, 0.2, True),
                                                       ("rms", False, None, 0.3, False), ("layer", False, 0.5, 0.0, False)])
def test_stack_and_loss_against_64_bits(norm, post, gate, drop, final):
    """Loss and every gradient. The layers' fp32 forwards and gradients are within 1e-5 of theirs; three of them and
    the norms between, whose factors are of order 1 here, keep the norm-wise distance under ten times that."""
    torch.manual_seed(7)
    rows, dim = 90, 24
    model = kan_amd.ResidualKAN([kan_amd.ChebyKANLayer(dim, dim, 4, init_scale=0.05) for _ in range(3)], dim, norm=norm,
                                post=post, gate=gate, scale=0.8, dropout=drop, final_norm=final).cuda()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "coeffs" not in name:
                p.add_(0.1 * torch.randn_like(p))
    x = torch.randn(rows, dim, device="cuda", requires_grad=True)
    targets = torch.randint(0, dim, (rows,), device="cuda")
    seed, offset = model.dropout_state.tolist()
    got = f.log_probs(model(x), targets)
    loss = -got.logp.mean() - 0.1 * got.entropy.mean()
    params = dict(model.named_parameters())
    grads = torch.autograd.grad(loss, [x, *params.values()])
    assert model.dropout_state.tolist() == [seed, offset + (3 if drop else 0)]

    keeps = [torch.from_numpy(orc.keep_mask(seed, offset + i, rows, dim, drop)).double() for i in range(3)] if drop else None
    x64 = x.detach().double().cpu().requires_grad_()
    p64 = {k: v.detach().double().cpu().requires_grad_() for k, v in params.items()}
    lp = torch.log_softmax(stack64(model, p64, x64, keeps), -1)
    want = -lp[torch.arange(rows), targets.cpu()].mean() + 0.1 * (lp.exp() * lp).sum(-1).mean()
    wants = torch.autograd.grad(want, [x64, *p64.values()])
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    for name, a, b in zip(["x", *params], grads, wants):
        assert ((a.cpu().double() - b).norm() <= 1e-4 * b.norm()), name


def test_eval_draws_nothing_and_state_travels():
    torch.manual_seed(1)
    model = kan_amd.ResidualKAN([kan_amd.ChebyKANLayer(16, 16, 3)], 16, dropout=0.5).cuda()
    x = torch.randn(8, 16, device="cuda")
    a, b = model(x), model(x)
    assert not torch.equal(a, b) and model.dropout_state[1].item() == 2
    other = kan_amd.ResidualKAN([kan_amd.ChebyKANLayer(16, 16, 3)], 16, dropout=0.5).cuda()
    other.load_state_dict(model.state_dict())
    assert torch.equal(model(x), other(x))
    model.eval()
    before = model.dropout_state.clone()
    assert torch.equal(model(x), model(x)) and torch.equal(model.dropout_state, before)


def test_refusals():
    layer = kan_amd.ChebyKANLayer(8, 9, 3)
    with pytest.raises(ValueError, match="maps 8 to 9"):
        kan_amd.ResidualKAN([layer], 8)
    with pytest.raises(ValueError, match="norm"):
        kan_amd.ResidualKAN([], 8, norm="batch")
    with pytest.raises(ValueError, match="probability"):
        kan_amd.ResidualKAN([], 8, dropout=1.5)


def test_example_trains_and_answers():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_residual
    finally:
        sys.path.pop(0)
    model, losses = train_residual.train(steps=30, rows=512, log=None)
    assert len(losses) == 30 and all(l == l for l in losses)
    assert all(torch.isfinite(p).all() for p in model.parameters())
    for got in train_residual.answer(model, 3):
        assert got.top_indices.shape == (1, 3) and (got.top_logp[:, :-1] >= got.top_logp[:, 1:]).all()
        assert 0 <= got.entropy.item() <= torch.log(torch.tensor(6.0)).item() + 1e-6


def test_single_rows_agree_with_the_batch():
    torch.manual_seed(3)
    blocks = [kan_amd.MixtureKANLayer(32, 32, 5, experts=8, top_k=2) for _ in range(2)]
    model = kan_amd.ResidualKAN(blocks, 32).cuda().eval()
    x = torch.randn(5, 32, device="cuda")
    with torch.no_grad():
        rows = torch.cat([model(x[r:r + 1]) for r in range(5)])
        assert ((rows - model(x)).norm() / rows.norm()).item() <= 1e-5
