"""A policy's memory: features of what an env has observed and done so far, from a stack of state space
blocks over the sequence operators (pnp_amd.seqops).

The shelf scene's observation holds positions, angles and fingers of one instant; what the gripper
pushed, how fast, and what it tried before is in the sequence.  ``HistoryEncoder`` maps a sequence of
tokens (normalised observation and previous action) to features that ``pnp_amd.tqc.TQC`` appends to the
observation (``TQCConfig(history=H)``):

* ``forward``  whole windows of the replay buffer, with gradients (training);
* ``step``     one token of every env against a carried state (rollout, evaluation), the projections
               in fp32, or in 8 bits with ``int8_weights()``.

A block: residual addition and RMS norm; projection to 2 x inner channels (u, z); causal convolution and
silu of u; projections of that to dt, B, C; selective scan gated by z; projection back.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import seqops


class _Block(nn.Module):
    def __init__(self, dim, inner, state, width, dt_rank):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(dim))
        self.in_proj = nn.Linear(dim, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, width).uniform_(-width ** -0.5, width ** -0.5))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, dt_rank + 2 * state, bias=False)
        self.dt_proj = nn.Linear(dt_rank, inner, bias=False)
        # softplus(dt_bias) spread over 0.001 .. 0.1 (log-uniform): decays from a few to a thousand tokens
        dt = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, state + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, dim, bias=False)
        self.split = (dt_rank, state, state)

    def _scan_inputs(self, x_dbl):
        dt, B, C = torch.split(x_dbl, self.split, dim=-1)
        return self.dt_proj(dt), -torch.exp(self.A_log), B, C

    def forward(self, h, stream, starts):
        y, stream = seqops.add_rms_norm(h, self.norm, stream)
        u, z = self.in_proj(y).chunk(2, dim=-1)
        u, _ = seqops.causal_conv(u, self.conv_weight, self.conv_bias, activation="silu", starts=starts)
        delta, A, B, C = self._scan_inputs(self.x_proj(u))
        o, _ = seqops.selective_scan(u, delta, A, B, C, D=self.D, z=z, delta_bias=self.dt_bias, starts=starts)
        return self.out_proj(o), stream

    def step(self, h, stream, state, reset, q=None):
        conv, ssm = state
        if q is None:
            y, stream = seqops.add_rms_norm(h, self.norm, stream)
            u, z = self.in_proj(y).chunk(2, dim=-1)
        else:
            y, scale, stream = seqops.add_rms_norm_q8(h, self.norm, stream)
            u, z = seqops.matmul_i8(y, scale, *q["in_proj"], out_dtype=h.dtype).chunk(2, dim=-1)
        u = seqops.causal_conv_step(u, conv, self.conv_weight, self.conv_bias, activation="silu", reset=reset)
        x_dbl = self.x_proj(u) if q is None else seqops.matmul_i8(*seqops.quantize_rows(u), *q["x_proj"], out_dtype=u.dtype)
        delta, A, B, C = self._scan_inputs(x_dbl)
        o = seqops.selective_scan_step(u, ssm, delta, A, B, C, D=self.D, z=z, delta_bias=self.dt_bias, reset=reset)
        h = self.out_proj(o) if q is None else seqops.matmul_i8(*seqops.quantize_rows(o), *q["out_proj"], out_dtype=o.dtype)
        return h, stream


class HistoryEncoder(nn.Module):
    """in_dim values a token -> dim features; ``layers`` blocks of ``expand * dim`` channels, ``state`` states a
    channel (up to 64), a convolution over ``width`` tokens (2 to 4).  Runs on a HIP device only, in its
    parameters' type (fp32, or ``.to(torch.bfloat16)`` / fp16: inputs and features are of that type then)."""

    def __init__(self, in_dim, dim=256, layers=1, state=16, width=4, expand=2, dt_rank=None):
        super().__init__()
        self.dim, self.inner, self.state, self.width = dim, expand * dim, state, width
        self.embed = nn.Linear(in_dim, dim)
        rank = dt_rank or max(1, math.ceil(dim / 16))
        self.blocks = nn.ModuleList(_Block(dim, self.inner, state, width, rank) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(dim))

    def forward(self, x, starts=None):
        """x [B, L, in_dim] -> features [B, L, dim]; starts [B, L] (uint8 or bool): tokens that begin an episode."""
        h, stream = self.embed(x), None
        for blk in self.blocks:
            h, stream = blk(h, stream, starts)
        return seqops.add_rms_norm(h, self.norm, stream)[0]

    def new_state(self, n):
        """The state of n envs that have seen nothing: per block (last tokens of the convolution, scan state)."""
        p = self.norm
        return [(torch.zeros(n, self.width - 1, self.inner, dtype=p.dtype, device=p.device),
                 torch.zeros(n, self.inner, self.state, dtype=torch.float32, device=p.device)) for _ in self.blocks]

    @torch.no_grad()
    def int8_weights(self):
        """The projections' weights in 8 bits with a scale per output channel, for ``step``; taken anew after the
        weights have changed."""
        return [{name: seqops.quantize_rows(getattr(blk, name).weight) for name in ("in_proj", "x_proj", "out_proj")}
                for blk in self.blocks]

    @torch.no_grad()
    def step(self, x, state, reset=None, int8=None):
        """One token of each of n envs: x [n, in_dim] -> features [n, dim]; ``state`` (``new_state``) advanced in
        place, begun anew for the envs that ``reset`` [n] marks.  int8: ``int8_weights()``, for products in 8 bits."""
        h, stream = F.linear(x, self.embed.weight, self.embed.bias), None
        for k, blk in enumerate(self.blocks):
            h, stream = blk.step(h, stream, state[k], reset, None if int8 is None else int8[k])
        return seqops.add_rms_norm(h, self.norm, stream)[0]
