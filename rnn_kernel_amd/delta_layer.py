"""A recurrent layer on the gated delta rule: projections, rule and output projection,
each one operator of the library.

* ``GatedDelta``: the module, for whole sequences (with gradients) and for one token
  of each of a batch of requests;
* ``python -m rnn_kernel_amd.delta_layer``: trains the layer to follow another one,
  then answers token by token from the trained states, and prints how far that is from
  the whole sequence.
"""
from __future__ import annotations

import argparse
import time
from typing import List, Optional, Tuple

import torch
from torch import nn

from .delta import gated_delta_rule, gated_delta_step
from .linear import Linear
from .train import AdamW, mse_loss


class GatedDelta(nn.Module):
    """y = x + W_o o, with o from the gated delta rule over

        q, k, v = silu(W_in x),   g = logsigmoid(W_g x + b_g),   beta = sigmoid(W_b x + b_b)

    q and k normalised, ``value_heads`` states of [key_dim, value_dim] per sequence; value
    head h reads key head h // (value_heads // key_heads).  All parameters are of one type,
    float32 or bfloat16; states are float32.  b_g starts at 3: a state loses a twentieth
    per token before anything is learnt."""

    def __init__(self, size: int, value_heads: int, key_dim: int, value_dim: int, key_heads: Optional[int] = None,
                 device=None, dtype=None) -> None:
        super().__init__()
        key_heads = value_heads if key_heads is None else key_heads
        if min(size, value_heads, key_heads, key_dim, value_dim) < 1 or value_heads % key_heads != 0:
            raise ValueError("GatedDelta: sizes must be >= 1 and value_heads a multiple of key_heads")
        self.size, self.key_heads, self.value_heads = size, key_heads, value_heads
        self.key_dim, self.value_dim = key_dim, value_dim
        like = dict(device=device, dtype=dtype)
        widths = 2 * key_heads * key_dim + value_heads * value_dim
        self.project = Linear(size, widths, bias=False, activation="silu", **like)
        self.decay = Linear(size, value_heads, activation="logsigmoid", **like)
        self.rate = Linear(size, value_heads, activation="sigmoid", **like)
        self.out = Linear(value_heads * value_dim, size, bias=False, **like)
        nn.init.constant_(self.decay.bias, 3.0)

    def new_states(self, count: int) -> torch.Tensor:
        """States of ``count`` sequences that have not begun."""
        return torch.zeros(count, self.value_heads, self.key_dim, self.value_dim, dtype=torch.float32,
                           device=self.out.weight.device)

    def _inputs(self, x: torch.Tensor):
        keys, values = self.key_heads * self.key_dim, self.value_heads * self.value_dim
        q, k, v = self.project(x).split([keys, keys, values], dim=-1)
        return (q.unflatten(-1, (self.key_heads, self.key_dim)), k.unflatten(-1, (self.key_heads, self.key_dim)),
                v.unflatten(-1, (self.value_heads, self.value_dim)), self.decay(x), self.rate(x))

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(y, state) of x [batch, tokens, size], as gated_delta_rule has state and lengths."""
        if x.dim() != 3 or x.size(-1) != self.size:
            raise ValueError(f"GatedDelta: x must have shape [batch, tokens, {self.size}]")
        o, state = gated_delta_rule(*self._inputs(x), state, normalize=True, lengths=lengths)
        return self.out(o.flatten(-2), residual=x), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, states: torch.Tensor, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y of x [requests, size], one token each; their ``states`` are updated in place, as
        gated_delta_step has states and slots."""
        if x.dim() != 2 or x.size(-1) != self.size:
            raise ValueError(f"GatedDelta: x must have shape [requests, {self.size}]")
        o = gated_delta_step(*self._inputs(x), states, slots=slots, normalize=True)
        return self.out(o.flatten(-2), residual=x)

    def extra_repr(self) -> str:
        return (f"size={self.size}, value_heads={self.value_heads}, key_heads={self.key_heads}, "
                f"key_dim={self.key_dim}, value_dim={self.value_dim}")


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


__all__: List[str] = ["GatedDelta", "main"]

if __name__ == "__main__":
    main()
