"""Grouped norm over the last dimension with a gate or an activation, on the HIP engine.

No counterpart in the reference, which normalizes whole rows (models/common.py:8-16): this is the
norm of each head's output in a multi-head recurrence, with the layer's SiLU gate applied in the
same pass.  Statistics are per row and group, never over positions, so it is causal.
"""

from . import _abi

_ACTIVATIONS = {None: 0, "silu": 1}


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, center=True, eps=1e-5):
    """y (x's shape and dtype) with, per row and group of C / groups <= 1024 channels,

        z = (x - mean) / sqrt(variance + eps) * weight + bias     (center=False: x / sqrt(mean(x^2) + eps) ...)
        y = z silu(gate) with a gate, silu(z) with activation="silu", else z

    x (..., C) float32, bfloat16 or float16; gate like x; weight, bias (C,).  float32 arithmetic;
    differentiable (once, reverse mode) in x, weight, bias and gate."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    if gate is not None and activation is not None:
        raise ValueError("a gate and an activation exclude each other")
    act = 2 if gate is not None else _ACTIVATIONS[activation]
    return _abi.host().gnorm(x, weight, bias, gate, int(groups), act, bool(center), float(eps))
