"""GatedDeltaMixer against a plain float64 composition on the CPU, its pieces and single tokens against one call.

Tolerances: the layer is two float32 GEMMs (sums of up to 96 terms, 2^-21 of the largest operand sum
each), the conv, the rule (2^-17 of its largest output) and the norm: 2^-15 of the output's largest
magnitude covers their sum; gradients pass the chain twice, 2^-14 of the largest entry of each."""

import pytest
import torch
import torch.nn.functional as F

from ssm_scan.delta_mixer import GatedDeltaMixer

pytestmark = pytest.mark.gpu


def plain(m, P, u):
    """The layer in float64 elementary operations, token by token; P: parameters by name."""
    B, L, _ = u.shape
    H, Hk, Dk, Dv = m.heads, m.key_heads, m.key_dim, m.value_dim
    p = u @ P["in_proj.weight"].t()
    mixed, z, dt, b = p.split([2 * m.d_keys + m.d_values, m.d_values, H, H], dim=-1)
    x = F.pad(mixed.transpose(1, 2), (m.d_conv - 1, 0))
    w = P["conv.weight"][:, 0]
    x = sum(w[:, j, None] * x[..., j:j + L] for j in range(m.d_conv)) + P["conv.bias"][:, None]
    q, k, v = (x * torch.sigmoid(x)).transpose(1, 2).split([m.d_keys, m.d_keys, m.d_values], dim=-1)
    head = torch.arange(H) // (H // Hk)
    q, k = (t.unflatten(-1, (Hk, Dk)) / (t.unflatten(-1, (Hk, Dk)).pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    q, k, v = q[:, :, head], k[:, :, head], v.unflatten(-1, (H, Dv))
    g, beta = -P["A_log"].exp() * F.softplus(dt + P["dt_bias"]), torch.sigmoid(b)
    S, o = u.new_zeros(B, H, Dk, Dv), []
    for t in range(L):
        S = S * g[:, t].exp()[..., None, None]
        y = v[:, t] - (k[:, t, :, :, None] * S).sum(-2)
        S = S + k[:, t, :, :, None] * (beta[:, t, :, None] * y)[:, :, None]
        o.append(Dk ** -0.5 * (q[:, t, :, :, None] * S).sum(-2))
    o = torch.stack(o, 1)
    o = (o / (o.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()).flatten(-2) * P["norm_weight"]
    return (o * z * torch.sigmoid(z)) @ P["out_proj.weight"].t()


def layer(dev, **kw):
    torch.manual_seed(0)
    return GatedDeltaMixer(**{**dict(d_model=96, heads=4, key_dim=32, value_dim=48, key_heads=2), **kw}).to(dev)


@pytest.mark.parametrize("L", [1, 70])
def test_forward_and_gradients_match_the_plain_layer(dev, L):
    m = layer(dev)
    u = torch.randn(2, L, 96, device=dev, requires_grad=True)
    do = torch.randn(2, L, 96, device=dev)
    out = m(u)
    got = torch.autograd.grad(out, [u] + list(m.parameters()), do)
    P = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    u64 = u.detach().double().cpu().requires_grad_()
    want_out = plain(m, P, u64)
    want = torch.autograd.grad(want_out, [u64] + list(P.values()), do.double().cpu())
    err = (out.detach().double().cpu() - want_out.detach()).abs().max().item()
    assert err <= 2.0 ** -15 * want_out.abs().max().item()
    for n, a, b in zip(["u"] + list(P), got, want):
        err = (a.double().cpu() - b).abs().max().item()
        assert err <= 2.0 ** -14 * b.abs().max().item(), (n, err / b.abs().max().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_and_single_tokens_continue_each_other(dev, dtype):
    """65, 1, 30 and 4 single tokens against one call (bf16: every activation is rounded, 2^-8 each, along a
    chain of six in either computation)."""
    m = layer(dev).to(dtype)
    m.A_log.data, m.dt_bias.data = m.A_log.data.float(), m.dt_bias.data.float()
    u = torch.randn(3, 100, 96, device=dev, dtype=dtype)
    with torch.no_grad():
        want = m(u)
        state, outs, t = m.init_state(3, dev, dtype), [], 0
        for n in (65, 1, 30, 1, 1, 1, 1):
            outs.append(m(u[:, t:t + n], state))
            t += n
    got = torch.cat(outs, 1)
    tol = 2.0 ** -15 if dtype == torch.float32 else 6 * 2.0 ** -8
    assert (got.double() - want.double()).abs().max().item() <= tol * want.abs().max().item()


def test_refusals(dev):
    with pytest.raises(ValueError, match="key heads"):
        GatedDeltaMixer(64, 4, 16, key_heads=3)
    with pytest.raises(ValueError, match="key_dim"):
        GatedDeltaMixer(64, 1, 160).to(dev)(torch.zeros(1, 3, 64, device=dev))
