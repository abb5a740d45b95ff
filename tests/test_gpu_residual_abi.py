"""The residual block's C entry points where their arguments go beyond what the Python front end passes."""
import pytest
import torch

from kan_amd import _lib

pytestmark = pytest.mark.gpu


def passes(rows, dim, gate_rows):
    """out, h, dx and dy of a block without a gate."""
    g = torch.Generator("cuda").manual_seed(dim)
    x, y, dout, dh = (torch.randn(rows, dim, device="cuda", generator=g) for _ in range(4))
    w = torch.rand(dim, device="cuda", generator=g)
    out, h, dx, dy = (torch.full_like(x, float("nan")) for _ in range(4))
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    desc = _lib.CkanResidualDesc(rows=rows, x_ld=dim, y_ld=dim, gate_ld=dim, dim=dim, gate_rows=gate_rows, eps=1e-6,
                                 scale=0.5)
    stats = torch.empty(lib.ckan_residual_stats_bytes(desc), dtype=torch.uint8, device="cuda")
    nbytes = lib.ckan_residual_workspace_bytes(desc)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    given = dict(x=x.data_ptr(), y=y.data_ptr(), post_weight=w.data_ptr(), next_weight=w.data_ptr(), stats=stats.data_ptr())
    _lib.check(lib.ckan_residual_forward(
        desc, _lib.CkanResidualBuffers(**given, out=out.data_ptr(), h=h.data_ptr()), stream))
    _lib.check(lib.ckan_residual_backward(
        desc, _lib.CkanResidualBuffers(**given, dout=dout.data_ptr(), dh=dh.data_ptr(), dout_ld=dim, dh_ld=dim,
                                       dx=dx.data_ptr(), dy=dy.data_ptr()), ws.data_ptr(), nbytes, stream))
    torch.cuda.synchronize()
    return out, h, dx, dy


@pytest.mark.parametrize("dim", [5, 40, 1000, 9000])
def test_a_null_gate_is_one_in_either_form(dim):
    for a, b in zip(passes(7, dim, 1), passes(7, dim, 0)):
        assert torch.equal(a, b) and torch.isfinite(a).all()
