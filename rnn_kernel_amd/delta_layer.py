"""A recurrent layer on the gated delta rule: projections, rule and output projection,
each one operator of the library.  ``GatedDelta`` is the module, for whole sequences
(with gradients) and for one token of each of a batch of requests.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import nn

from .delta import gated_delta_rule, gated_delta_step
from .linear import Linear


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


__all__: List[str] = ["GatedDelta"]
