"""The gated delta rule on the HIP engine: a recurrence with a matrix state per head.

No counterpart in the reference, whose scan has a diagonal state (models/scan.py:264-274); the
calls follow that scan's contract (h0 in, last state out, the state of a step updated in place).
Per batch row and value head, with S (Dk, Dv):

    S' = e^{g_t} S_{t-1}      u_t = beta_t (v_t - S'^T k_t)      S_t = S' + k_t u_t^T
    o_t = scale S_t^T q_t

``gated_delta_rule`` runs whole sequences (training, prefill; differentiable once in every tensor, in
reverse mode), ``gated_delta_step`` one token per stream.  Key heads may be fewer than value heads (value head h
reads key head h // (H // Hk)); their gradients are summed over the heads that share them.
Products run on the matrix cores over bf16 parts of the operands (one part for bf16 inputs, two
for fp16, three for float32 inputs and for the float32 intermediates); states,
decays, norms and sums are float32 or wider, and every sum runs in a fixed order.
"""

import torch

from . import _abi


def _scale(q, scale):
    if scale is None:
        return max(q.shape[-1], 1) ** -0.5 if q.dim() else 1.0   # no keys: the checks refuse them
    return float(scale)


def gated_delta_rule(q, k, v, g, beta, h0=None, scale=None, qk_norm=False, return_last_state=False):
    """o (B, L, H, Dv) in v's dtype; with return_last_state, (o, last (B, H, Dk, Dv) float32).

    q, k (B, L, Hk, Dk), Dk <= 128, Hk dividing H; v (B, L, H, Dv); all float32, bfloat16 or float16
    (read in place with any strides whose last one is 1).  g (B, L, H): log decays (<= 0; -inf forgets
    the state, as at a document's start); beta (B, L, H).  h0 (B, H, Dk, Dv): the state before the first
    token, zeros if None.  scale: Dk^-0.5 if None.  qk_norm divides q and k by sqrt(sum of squares + 1e-6)
    over Dk first.  An infinity or NaN reaches what the recurrence takes it to: outputs from its own token on
    (in v, those of its column), never those of earlier tokens, so that the end of a padded row may hold anything;
    an infinity may come out as NaN.  Gradients follow the adjoint likewise, but for one in g, which makes all of
    its 64 tokens' NaN."""
    scale = _scale(q, scale)
    if v.dim() == 4 and v.numel() == 0 and v.shape[2] and v.shape[3]:   # no token: the state passes through
        _abi.host().delta_checks(q, k, v, g, beta, h0)
        last = v.new_zeros((v.shape[0], v.shape[2], q.shape[-1], v.shape[3]), dtype=torch.float32) if h0 is None \
            else h0.float() * 1
        o = v * sum((t.sum() for t in (q, k, g, beta)), v.new_ones(())).to(v.dtype)   # in every operand's graph
        return (o, last) if return_last_state else o
    o, last = _abi.host().delta(q, k, v, g, beta, h0, scale, bool(qk_norm), bool(return_last_state))
    return (o, last) if return_last_state else o


def gated_delta_step(h, q, k, v, g, beta, scale=None, qk_norm=False):
    """One token per stream: o (B, H, Dv) in v's dtype; h (B, H, Dk, Dv), contiguous float32, is updated
    in place.  q, k (B, Hk, Dk), v (B, H, Dv), g and beta (B, H) as in gated_delta_rule.  Not differentiable: in
    grad mode, operands that require a gradient are refused."""
    scale = _scale(q, scale)
    return _abi.host().delta_step(h, q, k, v, g, beta, scale, bool(qk_norm))
