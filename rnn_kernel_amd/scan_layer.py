"""A recurrent layer on the selective scan: norm, projections, convolution, scan and output
projection, each one operator of the library.  ``SelectiveScan`` is the module, for whole
sequences (with gradients) and for one token of each of a batch of requests.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
from torch import nn

from .conv import MAX_CONV_WIDTH, MIN_CONV_WIDTH, causal_conv, causal_conv_step
from .linear import Linear, linear
from .norm import LayerNorm
from .scan import MAX_STATES, selective_scan, selective_step

State = Tuple[torch.Tensor, torch.Tensor]  # of the convolution and of the scan


class SelectiveScan(nn.Module):
    """y = x + W_o v, with u, z = W_in norm(x) of ``channels`` each and

        u' = silu(conv(u)),   d, B, C = W_x u',   dt = W_d d,   v = scan of u' with gate z

    (steps softplus(dt + b), ``states`` numbers of state per channel and ``groups`` of B and
    C).  The scan's A = -exp(A_log), skip and b are float32, whatever the module is cast to, the
    other parameters of one type, float32 or bfloat16.  A starts at -1 .. -states, steps at 0.001 to 0.1."""

    def __init__(self, size: int, channels: Optional[int] = None, states: int = 16, width: int = 4, groups: int = 1,
                 step_rank: Optional[int] = None, device=None, dtype=None) -> None:
        super().__init__()
        channels = 2 * size if channels is None else channels
        step_rank = max(1, size // 16) if step_rank is None else step_rank
        if min(size, channels, states, groups, step_rank) < 1 or channels % groups != 0:
            raise ValueError("SelectiveScan: sizes must be >= 1 and channels a multiple of groups")
        if states > MAX_STATES or not MIN_CONV_WIDTH <= width <= MAX_CONV_WIDTH:
            raise ValueError(f"SelectiveScan: states must be at most {MAX_STATES} and width in "
                             f"[{MIN_CONV_WIDTH}, {MAX_CONV_WIDTH}]")
        self.size, self.channels, self.states, self.width, self.groups = size, channels, states, width, groups
        self.step_rank = step_rank
        like = dict(device=device, dtype=dtype)
        self.norm = LayerNorm(size, **like)
        self.project = Linear(size, 2 * channels, bias=False, **like)
        bound = 1.0 / math.sqrt(width)
        self.conv_weight = nn.Parameter(torch.empty(channels, width, **like).uniform_(-bound, bound))
        self.conv_bias = nn.Parameter(torch.empty(channels, **like).uniform_(-bound, bound))
        self.inputs = Linear(channels, step_rank + 2 * groups * states, bias=False, **like)
        self.steps = Linear(step_rank, channels, bias=False, **like)
        self.out = Linear(channels, size, bias=False, **like)
        first = torch.exp(torch.rand(channels, device=device) * math.log(100.0) + math.log(1e-3))
        self.A_log = nn.Parameter(torch.arange(1, states + 1, dtype=torch.float32, device=device).log().repeat(channels, 1))
        self.skip = nn.Parameter(torch.ones(channels, dtype=torch.float32, device=device))
        self.step_bias = nn.Parameter((first + torch.log(-torch.expm1(-first))).to(torch.float32))

    def _apply(self, fn, recurse=True):
        # (what casts a module casts its parameters here: the scan's stay float32, wherever they go)
        wide = {id(t) for p in (self.A_log, self.skip, self.step_bias) for t in (p, p.grad) if t is not None}

        def keep(t):
            out = fn(t)
            return out if out.dtype == t.dtype or id(t) not in wide else t.to(out.device)

        return super()._apply(keep, recurse)

    def new_states(self, count: int) -> State:
        """States of ``count`` sequences that have not begun."""
        like = self.out.weight
        return (torch.zeros(count, self.width - 1, self.channels, dtype=like.dtype, device=like.device),
                torch.zeros(count, self.channels, self.states, dtype=torch.float32, device=like.device))

    def _scanned(self, u: torch.Tensor):
        of = self.groups * self.states
        d, B, C = self.inputs(u).split([self.step_rank, of, of], dim=-1)
        groups = (self.groups, self.states)
        return linear(d, self.steps.weight), -torch.exp(self.A_log), B.unflatten(-1, groups), C.unflatten(-1, groups)

    def forward(self, x: torch.Tensor, state: Optional[State] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, State]:
        """(y, state) of x [batch, tokens, size], as causal_conv and selective_scan have states
        and lengths; batch at most 65535 and tokens at most 2^20, as causal_conv takes them. Behind a
        row's end y is x, which has to be finite there for gradients of the weights."""
        if x.dim() != 3 or x.size(-1) != self.size:
            raise ValueError(f"SelectiveScan: x must have shape [batch, tokens, {self.size}]")
        before, h = (None, None) if state is None else state
        u, z = self.project(self.norm(x)).chunk(2, dim=-1)
        u, before = causal_conv(u, self.conv_weight, self.conv_bias, before, activation="silu", lengths=lengths)
        v, h = selective_scan(u, *self._scanned(u), h, skip=self.skip, gate=z, dt_bias=self.step_bias, softplus=True,
                              lengths=lengths)
        return self.out(v, residual=x), (before, h)

    @torch.no_grad()
    def step(self, x: torch.Tensor, states: State, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y of x [requests, size], one token each; their ``states`` are updated in place, as
        causal_conv_step and selective_step have states and slots."""
        if x.dim() != 2 or x.size(-1) != self.size:
            raise ValueError(f"SelectiveScan: x must have shape [requests, {self.size}]")
        u, z = self.project(self.norm(x)).chunk(2, dim=-1)
        u = causal_conv_step(u, states[0], self.conv_weight, self.conv_bias, activation="silu", slots=slots)
        v = selective_step(u, *self._scanned(u), states[1], skip=self.skip, gate=z, dt_bias=self.step_bias, softplus=True,
                           slots=slots)
        return self.out(v, residual=x)

    def extra_repr(self) -> str:
        return (f"size={self.size}, channels={self.channels}, states={self.states}, width={self.width}, groups={self.groups}, "
                f"step_rank={self.step_rank}")


__all__: List[str] = ["SelectiveScan"]
