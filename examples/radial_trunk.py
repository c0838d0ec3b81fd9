"""A radial network of the dense operators in front of the fused radial product, trained
for a few steps on synthetic edges.

    python examples/radial_trunk.py [--edges N] [--hidden H] [--blocks B] [--steps S]

Basis values go through ``RadialTrunk`` (linear layers with bias, SiLU and residual in
their epilogues, layer norms between them) to the hidden features of
``RadialUvuTensorProduct``, whose last affine layer is a ``Linear`` too.
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from ictc_o2_hp_b200 import Linear, RadialTrunk, RadialUvuTensorProduct, UvuTensorProduct


def main() -> int:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--edges", type=int, default=100_000)
    parser.add_argument("--hidden", type=int, default=64)
    parser.add_argument("--blocks", type=int, default=2)
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args()
    if not torch.cuda.is_available():
        print("needs a CUDA device")
        return 1
    device = torch.device("cuda")
    torch.manual_seed(0)
    tp = UvuTensorProduct(32, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    trunk = RadialTrunk(8, args.hidden, blocks=args.blocks).to(device)
    product = RadialUvuTensorProduct(tp, Linear(args.hidden, tp.weight_numel)).to(device)
    basis = torch.randn(args.edges, 8, device=device)
    left = torch.randn(args.edges, tp.input1_dimension, device=device)
    angular = torch.randn(args.edges, tp.input2_dimension, device=device)
    target = torch.randn(args.edges, tp.representation_dimension, device=device)
    params = [*trunk.parameters(), *product.parameters()]
    optimizer = torch.optim.Adam(params, lr=1e-3)
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for step in range(args.steps):
        if step == min(3, args.steps - 1):
            start.record()
        loss = (product(left, angular, trunk(basis)) - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        if step % 5 == 0:
            print(f"step {step:3d}  loss {loss.item():.6f}")
    stop.record()
    torch.cuda.synchronize()
    timed = args.steps - min(3, args.steps - 1)
    print(f"{start.elapsed_time(stop) / timed:.3f} ms a step, {args.edges} edges")
    return 0


if __name__ == "__main__":
    sys.exit(main())
