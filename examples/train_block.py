"""Trains one BidirectionalMamba block with group norm and an MLP with dropout in its fused form.

The task is synthetic: from a one-hot DNA sequence, predict at each position the base three to the left.

    python examples/train_block.py [--steps 200] [--length 512] [--width 128] [--dtype bf16]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from selectssm_b200 import BidirectionalMamba, dense_act  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=512)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--dtype", choices=["fp32", "bf16"], default="bf16")
    args = ap.parse_args()
    torch.manual_seed(0)
    dtype = torch.bfloat16 if args.dtype == "bf16" else torch.float32
    block = BidirectionalMamba(args.width, hidden_features=16, expansion_factor=2, norm_type="group", mlp_layer=True,
                               mlp_dropout_rate=0.1, fused_block=True).cuda()
    embed = torch.nn.Parameter(torch.randn(4, args.width, device="cuda"))
    head = torch.nn.Parameter(torch.randn(args.width, 4, device="cuda") / args.width ** 0.5)
    opt = torch.optim.Adam([*block.parameters(), embed, head], lr=2e-3)
    losses = []
    for step in range(args.steps):
        bases = torch.randint(0, 4, (args.batch, args.length), device="cuda")
        x = embed[bases].to(dtype)
        h = block(x, train=True, dropout_rng=(1234, 2 * step))  # a block uses two offsets a call
        logits = dense_act(h, head)
        target = torch.roll(bases, 3, dims=1)
        loss = torch.nn.functional.cross_entropy(logits[:, 3:].reshape(-1, 4).float(), target[:, 3:].reshape(-1))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if step % 50 == 0 or step == args.steps - 1:
            print(f"step {step}: loss {float(losses[-1]):.4f}")
    return [float(v) for v in (losses[0], losses[-1])]


if __name__ == "__main__":
    main()
