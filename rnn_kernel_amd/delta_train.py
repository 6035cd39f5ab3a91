"""``python -m rnn_kernel_amd.delta_train``: trains a gated delta-rule layer to follow
another one, then answers token by token from its states, and prints how far that is
from the whole sequence.
"""
from __future__ import annotations

import argparse
import time
from typing import List, Optional

import torch

from .delta_layer import GatedDelta
from .train import AdamW, mse_loss


def parse_args(argv: Optional[List[str]] = None) -> argparse.Namespace:
    p = argparse.ArgumentParser(description="Train a gated delta-rule layer and answer from it token by token.")
    p.add_argument("--size", type=int, default=256)
    p.add_argument("--heads", type=int, default=4)
    p.add_argument("--key-heads", type=int, default=2)
    p.add_argument("--head-dim", type=int, default=64)
    p.add_argument("--batch-size", type=int, default=8)
    p.add_argument("--seq-len", type=int, default=512)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--answer", type=int, default=32, help="tokens to answer after the prompt")
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--seed", type=int, default=42)
    p.add_argument("--device", type=str, default="cuda")
    return p.parse_args(argv)


def main(argv: Optional[List[str]] = None) -> dict:
    args = parse_args(argv)
    device = torch.device(args.device)
    if device.type != "cuda":
        raise RuntimeError("the layer runs on a GPU; --device must be a cuda/hip device")
    if not 1 <= args.answer < args.seq_len or args.steps < 1:
        raise ValueError("--answer must be in [1, seq-len) and --steps at least 1")
    torch.manual_seed(args.seed)

    def layer() -> GatedDelta:
        return GatedDelta(args.size, args.heads, args.head_dim, args.head_dim, args.key_heads, device=device)

    teacher, model = layer(), layer()
    optimizer = AdamW(model.parameters(), lr=args.lr, weight_decay=0.0)
    losses = []
    start = time.perf_counter()
    for _ in range(args.steps):
        x = torch.randn(args.batch_size, args.seq_len, args.size, device=device)
        with torch.no_grad():
            target = teacher(x)[0]
        loss = mse_loss(model(x)[0], target)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    seconds = time.perf_counter() - start
    print(f"trained {args.steps} steps of {args.batch_size} x {args.seq_len} tokens in {seconds:.2f} s: "
          f"loss {losses[0]:.5f} -> {losses[-1]:.5f}", flush=True)

    # the prompt at once, then the rest token by token, from states in a pool
    with torch.no_grad():
        whole, _ = model(x)
        prompt = args.seq_len - args.answer
        pool = model.new_states(args.batch_size + 1)
        slots = torch.arange(args.batch_size, 0, -1, dtype=torch.int32, device=device)
        y, state = model(x[:, :prompt])
        pool[slots.long()] = state
        out = [y]
        for t in range(prompt, args.seq_len):
            out.append(model.step(x[:, t], pool, slots)[:, None])
        error = ((torch.cat(out, dim=1) - whole).norm() / (whole - x).norm()).item()
    print(f"answered {args.answer} tokens of {args.batch_size} requests: {error:.2e} from the whole sequence", flush=True)
    return dict(losses=losses, error=error)


if __name__ == "__main__":
    main()
