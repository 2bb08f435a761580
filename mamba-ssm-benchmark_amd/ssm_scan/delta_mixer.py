"""A sequence mixer around the gated delta rule: what the Mamba mixer is around the selective scan.

No counterpart in the reference; the call follows its mixer (models/mamba.py:96-126: one module for
training, prefill in pieces with a carried state, and single tokens).  One projection gives the keys,
queries and values (which pass the causal conv and its SiLU, as the Mamba mixer's x does), the gate and
the two scalars per head:

    q, k, v = silu(conv(...))      g = -exp(A_log) softplus(dt + dt_bias)      beta = sigmoid(b)
    y = group_norm(gated_delta_rule(q, k, v, g, beta, qk_norm=True), heads, gate=z)      out_proj(y)

Everything between the two GEMMs but the two scalars runs in the engine's kernels; q, k, v and z are
read in place as parts of the projection.
"""

import math
from types import SimpleNamespace

import torch
import torch.nn as nn
import torch.nn.functional as F

from .conv import causal_conv1d
from .delta import gated_delta_rule, gated_delta_step
from .group_norm import group_norm
from .linear import linear, linear_act, plain_call


class GatedDeltaMixer(nn.Module):
    """(B, L, d_model) -> (B, L, d_model).  heads value heads of value_dim, key_heads (dividing heads; all
    by default) of key_dim <= 128.  With a state (init_state) the call continues the sequence and updates
    it, one token per call being the decode step.  A residual (B, L, d_model) is added to the output: in 16 bits
    (weights, u and residual of one type, no autocast, an nn.Linear without hooks) in the output projection's
    epilogue.  The states change in place, so such a call is inference: it runs without autograd whatever the grad
    mode, and its output has no graph."""

    def __init__(self, d_model, heads, key_dim, value_dim=None, key_heads=None, d_conv=4, dt_min=1e-3, dt_max=0.1):
        super().__init__()
        self.heads, self.key_heads = heads, key_heads or heads
        self.key_dim, self.value_dim, self.d_conv = key_dim, value_dim or key_dim, d_conv
        if heads % self.key_heads:
            raise ValueError(f"{heads} heads are not a multiple of {self.key_heads} key heads")
        self.d_keys, self.d_values = self.key_heads * key_dim, heads * self.value_dim
        d_mixed = 2 * self.d_keys + self.d_values
        self.in_proj = nn.Linear(d_model, d_mixed + self.d_values + 2 * heads, bias=False)
        self.conv = nn.Conv1d(d_mixed, d_mixed, d_conv, groups=d_mixed, bias=True)
        dt = torch.exp(torch.rand(heads) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))   # softplus^-1
        self.A_log = nn.Parameter(torch.log(torch.empty(heads).uniform_(1.0, 16.0)))
        self.norm_weight = nn.Parameter(torch.ones(self.d_values))
        self.out_proj = nn.Linear(self.d_values, d_model, bias=False)

    def init_state(self, batch, device, dtype=torch.float32):
        return SimpleNamespace(
            conv=torch.zeros(batch, 2 * self.d_keys + self.d_values, self.d_conv - 1, device=device, dtype=dtype),
            delta=torch.zeros(batch, self.heads, self.key_dim, self.value_dim, device=device))

    def _conv(self, x, state):
        if state is None or state.conv.dtype == x.dtype:
            return causal_conv1d(x, self.conv.weight, self.conv.bias, state=None if state is None else state.conv)
        previous = state.conv.to(x.dtype)   # a float32 state under autocast
        out = causal_conv1d(x, self.conv.weight, self.conv.bias, state=previous)
        state.conv.copy_(previous)
        return out

    def forward(self, u, state=None, residual=None):
        with torch.set_grad_enabled(torch.is_grad_enabled() and state is None):
            return self._forward(u, state, residual)

    def _forward(self, u, state, residual):
        mixed, z, dt, b = linear(self.in_proj, u).split(
            [2 * self.d_keys + self.d_values, self.d_values, self.heads, self.heads], dim=-1)
        mixed = self._conv(mixed, state)
        q, k, v = mixed.split([self.d_keys, self.d_keys, self.d_values], dim=-1)
        q, k = (t.unflatten(-1, (self.key_heads, self.key_dim)) for t in (q, k))
        v = v.unflatten(-1, (self.heads, self.value_dim))
        g = -torch.exp(self.A_log.float()) * F.softplus(dt.float() + self.dt_bias.float())
        beta = torch.sigmoid(b)
        if state is not None and u.shape[1] == 1:
            y = gated_delta_step(state.delta, q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], qk_norm=True).unsqueeze(1)
        else:
            y, last = gated_delta_rule(q, k, v, g, beta, h0=None if state is None else state.delta, qk_norm=True,
                                       return_last_state=True)
            if state is not None:
                state.delta.copy_(last)
        y = group_norm(y.flatten(-2), self.heads, self.norm_weight, gate=z, center=False)
        if residual is None:
            return linear(self.out_proj, y)
        if plain_call(self.out_proj, nn.Linear):
            w, bias = self.out_proj.weight, self.out_proj.bias
            if (w.dtype in (torch.bfloat16, torch.float16) and y.dtype == residual.dtype == w.dtype
                    and (bias is None or bias.dtype == w.dtype) and not torch.is_autocast_enabled(y.device.type)):
                return linear_act(y, w, bias, residual=residual)
        return residual + linear(self.out_proj, y)
