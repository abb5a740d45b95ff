"""Trains a classifier of residual ChebyKAN blocks, one of them a mixture, and answers single requests with it.

The classes are arcs of two interleaved spirals in the first two features; the others are noise.

Usage:  python examples/train_residual.py [--steps 300]
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import kan_amd  # noqa: E402
from kan_amd.functional import log_probs  # noqa: E402

WIDTH, CLASSES = 32, 6


def batch(rows: int):
    r = torch.rand(rows, device="cuda")
    arm = torch.randint(0, 2, (rows,), device="cuda")
    angle = 4.0 * r + 3.14159 * arm
    x = 0.3 * torch.randn(rows, 16, device="cuda")
    x[:, 0], x[:, 1] = 2 * r * torch.cos(angle), 2 * r * torch.sin(angle)
    return x, arm * (CLASSES // 2) + (r * (CLASSES // 2)).long().clamp(max=CLASSES // 2 - 1)


def build(dropout: float = 0.1) -> nn.Module:
    blocks = [kan_amd.ChebyKANLayer(WIDTH, WIDTH, 5), kan_amd.MixtureKANLayer(WIDTH, WIDTH, 5, experts=8, top_k=2),
              kan_amd.ChebyKANLayer(WIDTH, WIDTH, 5)]
    return nn.Sequential(kan_amd.ChebyKANLayer(16, WIDTH, 5), kan_amd.ResidualKAN(blocks, WIDTH, dropout=dropout, gate=0.5),
                         kan_amd.ChebyKANLayer(WIDTH, CLASSES, 3)).cuda()


def train(steps: int = 300, rows: int = 2048, seed: int = 0, log=print):
    """(model, losses): cross entropy with a small reward for entropy."""
    torch.manual_seed(seed)
    model = build()
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for step in range(steps):
        x, labels = batch(rows)
        got = log_probs(model(x), labels)
        loss = -got.logp.mean() - 0.01 * got.entropy.mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if log and (step % 50 == 0 or step == steps - 1):
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return model, losses


@torch.no_grad()
def answer(model, rows: int = 4):
    """Requests one at a time: each one's likeliest classes with their log probabilities."""
    model.eval()
    x, labels = batch(rows)
    return [log_probs(model(x[r:r + 1]), labels[r:r + 1], top=3) for r in range(rows)]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=300)
    model, _ = train(ap.parse_args().steps)
    for a in answer(model):
        print(f"label's log p {a.logp.item():7.3f}  entropy {a.entropy.item():.3f}  likeliest {a.top_indices[0].tolist()}")
