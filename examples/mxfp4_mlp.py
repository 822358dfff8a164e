"""Trains a residual MLP block in microscaled formats and serves it from its packed weights.

    PYTHONPATH=. python examples/mxfp4_mlp.py [--rows 4096] [--width 1024] [--steps 20]

Training runs the 4-bit layers on fp32 master weights; of every activation the graph keeps the 8-bit form.  Serving packs
the trained weights once and runs the same layers for whole batches and for single rows, with the residual in the last
layer's store."""

import argparse

import torch
import torch.nn as nn

from dimq_amd import DIMQMXFP4Linear, mx


class TrainBlock(nn.Module):
    def __init__(self, width: int, hidden: int) -> None:
        super().__init__()
        self.fc1, self.fc2 = mx.MXFP4TrainLinear(width, hidden), mx.MXFP4TrainLinear(hidden, width)

    def forward(self, x):
        return x + self.fc2(mx.gelu(self.fc1(x)))


class ServeBlock(nn.Module):
    def __init__(self, block: TrainBlock) -> None:
        super().__init__()
        self.fc1, self.fc2 = DIMQMXFP4Linear.from_linear(block.fc1), DIMQMXFP4Linear.from_linear(block.fc2)

    def forward(self, x):
        return self.fc2(self.fc1(x, activation="gelu"), residual=x)


def run(rows: int = 4096, width: int = 1024, steps: int = 20, seed: int = 0):
    """(losses, the trained block's output, the served block's, its output row by row) for one batch."""
    torch.manual_seed(seed)
    block = TrainBlock(width, 2 * width).cuda()
    optimiser = torch.optim.Adam(block.parameters(), lr=1e-3)
    x = torch.randn(rows, width, device="cuda", dtype=torch.bfloat16)
    turn = torch.linalg.qr(torch.randn(width, width)).Q.cuda().bfloat16()
    target = x + 0.5 * (x @ turn)  # what the block is to learn
    losses = []
    for _ in range(steps):
        loss = (block(x).float() - target.float()).square().mean()
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    served = ServeBlock(block)
    with torch.no_grad():
        return (torch.stack(losses).tolist(), block(x), served(x),
                torch.cat([served(x[i:i + 1]) for i in range(min(rows, 8))]))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    losses, trained, served, _ = run(a.rows, a.width, a.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
    print(f"trained and served outputs differ by at most {(trained.float() - served.float()).abs().max().item():.3g}")


if __name__ == "__main__":
    main()
