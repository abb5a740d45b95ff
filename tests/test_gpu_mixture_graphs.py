"""The mixture and orthogonalisation operators captured in a HIP graph: every replay, with other work between, is the eager result."""
import pytest
import torch

import kan_amd

pytestmark = pytest.mark.gpu
f = kan_amd.functional


def _route():
    bias = torch.linspace(-0.1, 0.1, 32, device="cuda")
    return torch.randn(300, 32, device="cuda"), lambda x: f.route(x, 4, score="sigmoid", bias=bias, groups=4, top_groups=2)


def _experts(rows, train):
    c = torch.randn(5, 40, 70, 6, device="cuda") / 40
    idx = torch.randint(-1, 5, (rows, 2), device="cuda")
    w = torch.rand(rows, 2, device="cuda")

    def call(x):
        if not train:
            return (f.kan_experts(x, c, idx, w),)
        # leaves of the call's own: a node made on another stream would draw that stream into the capture
        leaf, coeffs = x.detach().requires_grad_(), c.detach().requires_grad_()
        y = f.kan_experts(leaf, coeffs, idx, w)
        return (y.detach(),) + torch.autograd.grad(y, (leaf, coeffs), y.detach())

    return torch.randn(rows, 40, device="cuda"), call


def _orthogonal(shape, dtype, steps):
    return torch.randn(*shape, device="cuda").to(dtype), lambda x: (f.orthogonalize(x, steps=steps),)


def _muon(shape):
    g = torch.randn(*shape, device="cuda")

    def call(x):
        p, buf = x.clone(), torch.zeros_like(x)
        kan_amd.optim.muon_step_(p, g, buf, lr=0.1)
        return p, buf

    return torch.randn(*shape, device="cuda"), call


CASES = {
    "route": _route,
    "experts, few slots": lambda: _experts(9, False),
    "experts": lambda: _experts(400, False),
    "orthogonalize, small side": lambda: _orthogonal((2, 40, 200), torch.float32, 5),
    "orthogonalize, small side, runs": lambda: _orthogonal((2, 40, 200), torch.float32, 12),
    "orthogonalize, fp32": lambda: _orthogonal((130, 200), torch.float32, 5),
    "orthogonalize, two steps a pass": lambda: _orthogonal((260, 2100), torch.float32, 5),
    "orthogonalize, bf16": lambda: _orthogonal((200, 130), torch.bfloat16, 5),
    "muon": lambda: _muon((2, 20, 80, 5)),
    "experts, backward": lambda: _experts(400, True),
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
