"""The mixture layer's construction and refusals (no GPU)."""
import pytest
import torch

import kan_amd


def test_parameters_and_initialisation():
    torch.manual_seed(0)
    m = kan_amd.MixtureKANLayer(30, 20, 4, experts=6, top_k=2)
    assert {n: tuple(p.shape) for n, p in m.named_parameters()} == {"gate": (6, 30), "cheby_coeffs": (6, 30, 20, 5)}
    assert abs(m.cheby_coeffs.std().item() * 150 - 1) < 0.05
    assert set(m.state_dict()) == {"gate", "cheby_coeffs"}
    assert m.get_analytical_form()["experts"] == 6
    assert "experts=6" in repr(m)


@pytest.mark.parametrize("kw,match", [
    (dict(score="relu"), "score"), (dict(compute="fp16"), "compute"), (dict(top_k=9), "top_k"),
    (dict(groups=3), "groups"), (dict(groups=2, top_groups=1, top_k=5), "top_k"), (dict(degree=0), "degree"),
    (dict(degree=17), "degree"),
])
def test_refusals(kw, match):
    args = dict(input_dim=4, output_dim=3, degree=2, experts=8, top_k=2)
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        kan_amd.MixtureKANLayer(**args)


def test_balance_needs_its_bias_and_a_forward():
    with pytest.raises(RuntimeError, match="balance=True"):
        kan_amd.MixtureKANLayer(4, 3, 2, 4).update_balance()
    with pytest.raises(RuntimeError, match="forward"):
        kan_amd.MixtureKANLayer(4, 3, 2, 4, balance=True).update_balance()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm device"):
        kan_amd.MixtureKANLayer(4, 3, 2, 4)(torch.zeros(2, 4))
