"""Forward-mode tangents are refused, not dropped (checked before the device is, so no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import kan_amd

f = kan_amd.functional
IDX = torch.zeros(3, 1, dtype=torch.int64)


def _calls():
    x, c, e, w = torch.randn(3, 4), torch.randn(4, 5, 3), torch.randn(2, 4, 5, 3), torch.ones(3, 1)
    return {
        "route": (lambda l: f.route(l, 1), (x,)),
        "kan_experts": (lambda *a: f.kan_experts(a[0], a[1], IDX, a[2]), (x, e, w)),
        "orthogonalize": (f.orthogonalize, (x,)),
        "chebykan": (f.chebykan, (x, c)),
        "family_kan": (lambda a, b: f.family_kan(a, b, None), (x, c)),
        "jacobian": (lambda a, b: f.jacobian(a, b, None), (x, c)),
    }


@pytest.mark.parametrize("name,which", [("route", 0), ("kan_experts", 0), ("kan_experts", 1), ("kan_experts", 2),
                                        ("orthogonalize", 0), ("chebykan", 0), ("chebykan", 1), ("family_kan", 0),
                                        ("family_kan", 1), ("jacobian", 0), ("jacobian", 1)])
def test_tangents_are_refused(name, which):
    call, args = _calls()[name]
    with fwad.dual_level():
        dual = [fwad.make_dual(a, torch.ones_like(a)) if k == which else a for k, a in enumerate(args)]
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*dual)
        with pytest.raises(RuntimeError) as plain:  # without one the call gets to the device check
            call(*args)
    assert "forward-mode" not in str(plain.value)


def test_a_layer_refuses_them():
    layer = kan_amd.ChebyKANLayer(4, 5, 2)
    mixture = kan_amd.MixtureKANLayer(4, 5, 2, experts=3)
    for p in list(layer.parameters()) + list(mixture.parameters()):
        p.requires_grad_(False)
    x = torch.randn(3, 4)
    with fwad.dual_level():
        for m in (layer, mixture):
            with pytest.raises(RuntimeError, match="forward-mode"):
                m(fwad.make_dual(x, torch.ones_like(x)))
