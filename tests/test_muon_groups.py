"""What Muon takes as parameters, at construction and later (no GPU)."""
import pytest
import torch

import kan_amd


def test_groups_added_later_are_checked():
    opt = kan_amd.optim.Muon([torch.nn.Parameter(torch.zeros(4, 5))])
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(opt.param_groups) == 1  # the refused group is not kept
    opt.add_param_group({"params": torch.nn.Parameter(torch.zeros(3, 4, 5)), "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [0.02, 0.5]
    with pytest.raises(ValueError, match="matrices"):
        kan_amd.optim.Muon([torch.nn.Parameter(torch.zeros(2, 2)), torch.nn.Parameter(torch.zeros(()))])
