"""The residual-block, dropout, log-probability and few-row mixture operators captured in a HIP graph, on other streams and side by
side: every replay, with other work between, is the eager result."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def _residual(shape, dtype, drop, train):
    dim = shape[-1]
    w = [torch.rand(dim, device="cuda") + 0.5 for _ in range(4)]
    y0 = torch.randn(*shape, device="cuda").to(dtype)

    def call(x):
        # leaves of the call's own: a node made on another stream would draw that stream into the capture
        leaves = [t.detach().requires_grad_(train) for t in (x, y0, *w)]
        out, h = f.residual_norm(leaves[0], leaves[1], norm="layer", post_weight=leaves[2], gate=leaves[3],
                                 next_weight=leaves[4], next_bias=leaves[5], dropout=drop, dropout_state=11)
        if not train:
            return out, h
        return (out.detach(), h.detach()) + torch.autograd.grad((out, h), leaves, (x, y0))

    return torch.randn(*shape, device="cuda").to(dtype), call


def _dropout(shape, dtype):
    def call(x):
        leaf = x.detach().requires_grad_()
        y = f.dropout(leaf, 0.3, 5, 2)
        return (y.detach(),) + torch.autograd.grad(y, leaf, x)

    return torch.randn(*shape, device="cuda").to(dtype), call


def _log_probs(rows, classes, top, train):
    t = torch.randint(0, classes, (rows,), device="cuda")
    up = torch.randn(rows, device="cuda")

    def call(x):
        leaf = x.detach().requires_grad_(train)
        got = f.log_probs(leaf, t, top=top)
        out = tuple(v.detach() for v in got if v is not None)
        return out + torch.autograd.grad((got.logp, got.entropy), leaf, (up, up)) if train else out

    return torch.randn(rows, classes, device="cuda"), call


def _mixture(rows, in_dim, out_dim, experts):
    g = torch.randn(experts, in_dim, device="cuda")
    c = torch.randn(experts, in_dim, out_dim, 6, device="cuda") / in_dim

    def call(x):
        with torch.no_grad():
            return f.kan_mixture(x, g, c, 2)

    return torch.randn(rows, in_dim, device="cuda"), call


CASES = {
    "residual, team": lambda: _residual((50, 300), torch.float32, 0.2, True),
    "residual, bf16": lambda: _residual((700, 64), torch.bfloat16, 0.0, True),
    "residual, wide": lambda: _residual((6, 9000), torch.float32, 0.2, True),
    "residual, forward": lambda: _residual((1, 2048), torch.bfloat16, 0.0, False),
    "dropout": lambda: _dropout((77, 130), torch.bfloat16),
    "log_probs, team": lambda: _log_probs(200, 70, 4, True),
    "log_probs, block": lambda: _log_probs(600, 3000, 4, True),
    "log_probs, long rows": lambda: _log_probs(600, 5000, 4, True),
    "log_probs, parts": lambda: _log_probs(2, 50000, 20, True),
    "mixture, one row": lambda: _mixture(1, 300, 200, 8),
    "mixture, few rows": lambda: _mixture(7, 300, 200, 8),
    "mixture, stream": lambda: _mixture(30, 300, 200, 8),
    "mixture, large gate": lambda: _mixture(3, 700, 40, 200),
}


@pytest.mark.parametrize("name", list(CASES))
def test_replays(name):
    torch.manual_seed(len(name))
    x, call = CASES[name]()
    fixed = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(fixed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(fixed)
    for k in range(4):
        other = torch.randn_like(x, dtype=torch.float32).to(x.dtype) if k else x
        want = [v.detach().clone() for v in call(other)]
        fixed.copy_(other)
        torch.cuda.synchronize()
        graph.replay()
        noise = torch.randn(1 << 20, device="cuda").sort()  # eager work that takes and frees memory
        del noise
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.parametrize("name", list(CASES))
def test_two_streams_at_once(name):
    torch.manual_seed(len(name))
    x, call = CASES[name]()
    others = [torch.randn_like(x, dtype=torch.float32).to(x.dtype) for _ in range(2)]
    want = [[v.detach().clone() for v in call(o)] for o in others]
    streams = [torch.cuda.Stream() for _ in others]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = call(others[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_a_captured_step_draws_new_masks_at_every_replay():
    torch.manual_seed(0)
    state = torch.tensor([123, 0], device="cuda")
    x = torch.ones(64, 96, device="cuda")

    def step():
        leaf = x.detach().requires_grad_()
        y = f.dropout(leaf, 0.4, state)
        state[1:].add_(1)  # the gradient still belongs to the mask that was drawn
        return y.detach(), torch.autograd.grad(y, leaf, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    first = int(state[1])
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = f.dropout(x, 0.4, 123, first + k)
        assert torch.equal(y, want) and torch.equal(g, want)
    assert int(state[1]) == first + 4
