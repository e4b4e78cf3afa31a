"""Fine-tunes the experts of a 16-bit MoE block on a synthetic target and then
decodes with it: router -> dispatch -> grouped products -> combine, with the
shared expert, forward and backward, all on the package's kernels.

    python examples/moe_finetune.py [--tokens 1024] [--steps 20]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "sen-mlx_b200"))
import senmoe  # noqa: E402
from senmoe.block16 import Moe16, Moe16Weights  # noqa: E402


def make_block(hidden, intermediate, experts, top_k, shared, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, fan_in):
        return (torch.randn(*shape, generator=g, device=device) / fan_in ** 0.5).to(torch.bfloat16)
    w = Moe16Weights(normal(experts, hidden, fan_in=hidden), normal(experts, 2 * intermediate, hidden, fan_in=hidden),
                     normal(experts, hidden, intermediate, fan_in=intermediate),
                     normal(2 * shared, hidden, fan_in=hidden), normal(hidden, shared, fan_in=shared))
    return Moe16(w, top_k)


def train(block, teacher, x, steps, lr):
    """Plain gradient steps on fp32 copies of the weights; the loss of each.
    A step whose kernels gave up a wait raises before it is taken."""
    names = ("gate_up", "down", "shared_gate_up", "shared_down")
    master = {n: getattr(block.w, n).float() for n in names}
    target = teacher.forward(x).float()
    losses = []
    for _ in range(steps):
        h, saved = block.forward(x, train=True)
        off = h.float() - target
        losses.append(float(off.square().mean()))
        _, grads = block.backward((off * (2.0 / x.shape[0])).to(h.dtype), saved)
        senmoe.linear_check()
        for n in names:
            master[n] -= lr * grads[n].float()
            getattr(block.w, n).copy_(master[n])
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--intermediate", type=int, default=768)
    ap.add_argument("--experts", type=int, default=32)
    ap.add_argument("--top-k", type=int, default=4)
    ap.add_argument("--shared", type=int, default=512)
    a = ap.parse_args()
    sizes = (a.hidden, a.intermediate, a.experts, a.top_k, a.shared)
    block, teacher = make_block(*sizes, seed=0), make_block(*sizes, seed=1)
    teacher.w.router = block.w.router
    x = torch.randn(a.tokens, a.hidden, device="cuda").to(torch.bfloat16)
    losses = train(block, teacher, x, a.steps, lr=0.02)
    print("loss by step:", " ".join(f"{v:.4f}" for v in losses))
    # decode: one token at a time through the few-row products
    whole = block.forward(x[:8]).float()
    steps = torch.cat([block.forward(x[t:t + 1]) for t in range(8)]).float()
    print(f"8 tokens decoded one by one against together: relative L2 {float((steps - whole).norm() / whole.norm()):.2e}")


if __name__ == "__main__":
    main()
