"""Float64 restatements, on the CPU, of what a language model does around its mixers: the token embedding, the norm
with the residual's addition and its 8-bit rows, the linear layer with its epilogue, the draw of the next token.

Gradients are written out by hand.  Every function takes tensors of any type and device and returns float64 ones.
"""

import math

import numpy as np
import torch

TOP8 = 448.0   # the largest e4m3 value


def wide(t):
    return None if t is None else t.detach().double().cpu()


def embedding(tokens, weight, scale=1.0, dout=None):
    """out; with dout, (out, dweight, the sum of the magnitudes that dweight adds)."""
    tokens, w = tokens.detach().cpu().reshape(-1).long(), wide(weight)
    there = (tokens >= 0) & (tokens < w.shape[0])
    out = torch.zeros(tokens.numel(), w.shape[1], dtype=torch.float64)
    out[there] = scale * w[tokens[there]]
    if dout is None:
        return out
    d = wide(dout).reshape(out.shape)
    dw, mag = torch.zeros_like(w), torch.zeros_like(w)
    dw.index_add_(0, tokens[there], scale * d[there])
    mag.index_add_(0, tokens[there], abs(scale) * d[there].abs())
    return out, dw, mag


def norm(s, weight, eps=1e-5, dy=None, ds=None):
    """y of rows s; with dy, (y, the gradient of s, of weight, and the magnitudes that the latter adds)."""
    s, w = wide(s), wide(weight)
    r = (s.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    y = s * r * w
    if dy is None:
        return y
    dy = wide(dy)
    h = dy * w
    d = r * (h - s * r * r * (h * s).mean(-1, keepdim=True))
    if ds is not None:
        d = d + wide(ds)
    terms = (dy * s * r).reshape(-1, s.shape[-1])
    return y, d, terms.sum(0), terms.abs().sum(0)


def rows8_scale(y):
    """The scale of rows y: NaNs do not count."""
    top = torch.nan_to_num(y.abs(), nan=0.0, posinf=math.inf).amax(-1)
    return torch.where(top > 0, top / TOP8, torch.ones_like(top))


def act(z, name):
    """(act(z), act'(z))"""
    if name == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    if name == "gelu":
        g = torch.special.ndtr(z)
        return z * g, g + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def linear(x, weight, bias=None, activation=None, residual=None, dy=None):
    """dict: y, z, the sum of magnitudes of z's terms; with dy also dz, dx, dw, dbias, dresidual."""
    x, w = wide(x), wide(weight)
    lead, x = x.shape[:-1], x.reshape(-1, x.shape[-1])
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, mag = z + wide(bias), mag + wide(bias).abs()
    y, slope = act(z, activation)
    if residual is not None:
        y = y + wide(residual).reshape(y.shape)
    res = dict(y=y.reshape(lead + y.shape[-1:]), z=z, mag=mag, slope=slope)
    if dy is not None:
        dy = wide(dy).reshape(z.shape)
        dz = dy * slope
        res.update(dz=dz, dx=dz @ w, dw=dz.t() @ x, dbias=dz.sum(0), dresidual=dy, x=x, w=w, dy=dy)
    return res


def sample(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(tokens, log probabilities) of rows of logits (B, V), as int64 and float64 arrays."""
    logits, u = wide(logits).numpy(), wide(u).numpy()

    def of(v, b, off):
        return off if v is None else float(v[b]) if isinstance(v, torch.Tensor) else float(v)

    tokens, logprobs = [], []
    for b, row in enumerate(logits):
        T, k, p, m = of(temperature, b, 1.0), of(top_k, b, 0), of(top_p, b, 1.0), of(min_p, b, 0.0)
        if np.isnan(row).any() or not (row > -np.inf).any():
            tokens.append(-1)
            logprobs.append(math.nan)
            continue
        order = np.lexsort((np.arange(row.size), -row))
        if not T > 0:
            order, T = order[:1], 1.0
        elif k >= 1:
            order = order[:int(k)]
        top = row[order[0]]
        with np.errstate(invalid="ignore"):
            w = np.where(row[order] == top, 1.0, np.exp((row[order] - top) / T))
        if p < 1:
            reach = int(np.argmax(np.cumsum(w) >= p * w.sum())) + 1
            order, w = order[:reach], w[:reach]
        keep = w >= m
        keep[0] = True
        order, w = order[keep], w[keep]
        back = np.argsort(order)
        order, w = order[back], w[back]
        at = min(int(np.searchsorted(np.cumsum(w), u[b] * w.sum(), side="right")), len(w) - 1)
        while w[at] == 0 and at > 0:   # a u of 1: the last with any mass
            at -= 1
        tokens.append(int(order[at]))
        logprobs.append(math.log(w[at] / w.sum()))
    return np.array(tokens), np.array(logprobs)
