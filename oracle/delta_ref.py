"""Float64 oracles of the gated delta rule and the grouped norm, on the CPU: the recurrence token by
token with its hand-written adjoint, and the norm's formulas."""

import torch

NORM_EPS = 1e-6


def _unit(x, qk_norm):
    n = (x.pow(2).sum(-1, keepdim=True) + NORM_EPS).sqrt() if qk_norm else torch.ones_like(x[..., :1])
    return x / n, n


def delta(q, k, v, g, beta, h0=None, scale=None, qk_norm=False, dout=None, dlast=None):
    """(o, last), or with dout and/or dlast (o, last, gradients by name).  Shapes as gated_delta_rule's."""
    q, k, v, g, beta = (t.detach().double().cpu() for t in (q, k, v, g, beta))
    B, L, H, Dv = v.shape
    Hk, Dk = q.shape[2:]
    scale = Dk ** -0.5 if scale is None else scale
    (qn, nq), (kn, nk) = _unit(q, qk_norm), _unit(k, qk_norm)
    head = torch.arange(H) // (H // Hk)
    Q, K = qn[:, :, head], kn[:, :, head]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    o, y, before, after = torch.zeros_like(v), torch.zeros_like(v), [], []
    for t in range(L):
        S = S * g[:, t].exp()[..., None, None]
        before.append(S)
        y[:, t] = v[:, t] - torch.einsum("bhk,bhkv->bhv", K[:, t], S)
        S = S + K[:, t, :, :, None] * (beta[:, t, :, None] * y[:, t])[:, :, None]
        after.append(S)
        o[:, t] = scale * torch.einsum("bhk,bhkv->bhv", Q[:, t], S)
    if dout is None and dlast is None:
        return o, S
    dout = torch.zeros_like(o) if dout is None else dout.detach().double().cpu()
    D = torch.zeros_like(S) if dlast is None else dlast.detach().double().cpu()
    dQ, dK, dv, dg, db = (torch.zeros_like(t) for t in (Q, K, v, g, beta))
    for t in reversed(range(L)):
        b = beta[:, t, :, None]
        do = scale * dout[:, t]
        dQ[:, t] = torch.einsum("bhkv,bhv->bhk", after[t], do)
        D = D + Q[:, t, :, :, None] * do[:, :, None]
        du = torch.einsum("bhk,bhkv->bhv", K[:, t], D)
        db[:, t] = (du * y[:, t]).sum(-1)
        dv[:, t] = b * du
        dK[:, t] = torch.einsum("bhkv,bhv->bhk", D, b * y[:, t]) - torch.einsum("bhkv,bhv->bhk", before[t], b * du)
        D = D - K[:, t, :, :, None] * (b * du)[:, :, None]
        dg[:, t] = (D * before[t]).sum((-1, -2))
        D = D * g[:, t].exp()[..., None, None]

    def back(d, unit, n):
        d = d.unflatten(2, (Hk, H // Hk)).sum(3)
        return (d - unit * (unit * d).sum(-1, keepdim=True)) / n if qk_norm else d

    def whole(d, n):   # the largest entry of what the norm's gradient projects
        return (d.unflatten(2, (Hk, H // Hk)).sum(3) / n).abs().max().item()

    return o, S, dict(q=back(dQ, qn, nq), k=back(dK, kn, nk), v=dv, g=dg, beta=db, h0=D,
                      size=dict(q=whole(dQ, nq), k=whole(dK, nk)))


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, center=True, eps=1e-5, dout=None):
    """y, or with dout (y, gradients by name)."""
    shape, C = x.shape, x.shape[-1]
    x = x.detach().double().cpu().reshape(-1, groups, C // groups)
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    x = x - x.mean(-1, keepdim=True) if center else x
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x * r).reshape(-1, C)
    z = xh * w + b
    a = z if gate is None else gate.detach().double().cpu().reshape(-1, C)
    s = torch.sigmoid(a)
    ds = s * (1 + a * (1 - s))
    y = z * a * s if gate is not None else a * s if activation else z
    if dout is None:
        return y.reshape(shape)
    dy = dout.detach().double().cpu().reshape(-1, C)
    dz = dy * (a * s if gate is not None else ds if activation else 1.0)
    h, xg = (dz * w).reshape(x.shape), xh.reshape(x.shape)
    dx = h - xg * (h * xg).mean(-1, keepdim=True) - (h.mean(-1, keepdim=True) if center else 0.0)
    return y.reshape(shape), dict(x=(dx * r).reshape(shape), weight=(dz * xh).sum(0), bias=dz.sum(0),
                                  gate=(dy * z * ds).reshape(shape))
