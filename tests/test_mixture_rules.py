"""Which calls the few-row mixture takes (host rule, no GPU): each limit from both sides."""
import pytest

from kan_amd import _lib


def few(rows, experts, top_k, in_dim, out_dim, degree, coeff_bf16=0):
    desc = _lib.CkanMixtureDesc(rows, experts, top_k, in_dim, out_dim, degree, 0, 1, 1, 1, 0, 0, coeff_bf16, 1.0)
    taken = _lib.load().ckan_mixture_few(desc)
    assert (_lib.load().ckan_mixture_workspace_bytes(desc) > 0) == bool(taken)
    return taken


@pytest.mark.parametrize("args,taken", [
    ((0, 8, 2, 64, 64, 4), 0), ((1, 8, 2, 64, 64, 4), 1),
    ((512, 32, 2, 64, 64, 4), 1), ((513, 32, 2, 64, 64, 4), 0),   # 1024 slots
    ((255, 8, 2, 64, 64, 4), 1), ((256, 8, 2, 64, 64, 4), 0),     # 64 an expert
    ((63, 1, 1, 64, 64, 4), 1), ((64, 1, 1, 64, 64, 4), 0),
])
def test_slots(args, taken):
    assert few(*args) == taken


# fp32 coefficients of degree 9 and more, from 9 rows on, below 8 slots an expert, 2^25 of them and more
@pytest.mark.parametrize("args,taken", [
    ((9, 12, 3, 300, 700, 16), 0), ((8, 12, 3, 300, 700, 16), 1), ((31, 12, 3, 300, 700, 16), 0),
    ((32, 12, 3, 300, 700, 16), 1), ((9, 12, 3, 300, 700, 16, 1), 1), ((9, 12, 3, 300, 700, 8), 1),
    ((16, 8, 2, 512, 512, 16), 0), ((16, 8, 2, 512, 512, 15), 0), ((16, 8, 2, 512, 512, 14), 1),
    ((16, 64, 2, 512, 512, 9), 0), ((16, 64, 2, 200, 200, 9), 1),
    ((8, 128, 8, 256, 256, 16), 1), ((8, 128, 9, 256, 256, 16), 0), ((8, 128, 9, 300, 300, 16), 1),  # 64 slots, experts of 5 MiB
])
def test_high_degrees(args, taken):
    assert few(*args) == taken


def test_a_bf16_layer_casts_no_coefficients_for_few_rows():
    """The layer's own count of few rows has no limit for high degrees."""
    import torch
    import kan_amd
    with torch.device("meta"), torch.no_grad():
        for degree in (8, 16):
            layer = kan_amd.MixtureKANLayer(300, 700, degree, experts=12, top_k=3, compute="bf16")
            assert [layer._few(torch.zeros(rows, 300)) for rows in (1, 9, 255, 256)] == [True, True, True, False]
