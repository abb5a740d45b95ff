"""Trains a mixture of ChebyKAN experts with Muon and serves single rows from it.

The target is a piecewise function: which of four smooth maps applies depends on
where the row lies, so a gate that sends regions to experts has something to find.

Usage:  python examples/train_mixture.py [--steps 200] [--compute bf16]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import kan_amd  # noqa: E402


def target(x: torch.Tensor) -> torch.Tensor:
    region = (x[:, 0] > 0).long() * 2 + (x[:, 1] > 0).long()
    u = x[:, 2:10]
    pieces = torch.stack([torch.sin(2 * u), u * u - 1, torch.tanh(3 * u), torch.cos(2 * u) * u], 0)
    return pieces[region, torch.arange(len(x), device=x.device)]


def train(steps: int = 200, rows: int = 4096, compute: str = "fp32", seed: int = 0, log=print):
    """(model, losses): the gate by Adam, the experts' coefficients by Muon."""
    torch.manual_seed(seed)
    model = kan_amd.MixtureKANLayer(16, 8, degree=6, experts=8, top_k=2, score="sigmoid", balance=True,
                                    compute=compute).cuda()
    experts = kan_amd.optim.Muon([model.cheby_coeffs], lr=0.02)
    gate = kan_amd.optim.Adam([model.gate], lr=0.01)
    losses = []
    for step in range(steps):
        x = torch.randn(rows, 16, device="cuda")
        loss = torch.nn.functional.mse_loss(model(x), target(x))
        experts.zero_grad()
        gate.zero_grad()
        loss.backward()
        experts.step()
        gate.step()
        model.update_balance()
        losses.append(loss.item())
        if log and (step % 20 == 0 or step == steps - 1):
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return model, losses


@torch.no_grad()
def serve(model, rows: int = 4) -> torch.Tensor:
    """Rows one at a time, as requests come in."""
    x = torch.randn(rows, 16, device="cuda")
    return torch.cat([model(x[r:r + 1]) for r in range(rows)]) - model(x)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--compute", choices=("fp32", "bf16"), default="fp32")
    a = ap.parse_args()
    model, _ = train(a.steps, compute=a.compute)
    print(f"single rows against the batch: largest difference {serve(model).abs().max().item():.1e}")
