"""What the gated delta rule's arithmetic keeps where the terms of an output cancel.

Outputs in 16 bits are half a step of their value off (eps / 2); everything before is float32 or bf16 parts of
24 bits, so that terms of size 1 may leave 2^-21 beside it: two exponentials and their differences (2^-23 each
at most), two products and a sum (2^-24 each)."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan
from test_gpu_delta import close, make

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
TERMS = 2.0 ** -21


def run(dev, io, q, k, v, g, beta, h0=None):
    """One batch row of many heads, scale 1, against the oracle; the last token's output."""
    a = dict(q=q.to(io), k=k.to(io), v=v.to(io), g=g, beta=beta)
    o = ssm_scan.gated_delta_rule(**{n: t.to(dev) for n, t in a.items()}, h0=None if h0 is None else h0.to(dev), scale=1.0)
    want, _ = delta_ref.delta(**a, h0=h0, scale=1.0)
    tol = torch.finfo(io).eps / 2 * want.abs() + TERMS
    err = (o.double().cpu() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    assert want[:, -1].abs().max() < 2.0 ** -11   # the terms of size 1 have cancelled


@pytest.mark.parametrize("io", [BF16, F16])
def test_rows_of_the_state_that_cancel(dev, io):
    """o = S_0 + S_1 with rows x and -x (1 - r 2^-12)."""
    H, Dv = 3, 40
    x, r = torch.rand(2, H, Dv, generator=torch.Generator().manual_seed(0))
    h0 = torch.stack([0.5 + x / 2, -(0.5 + x / 2) * (1 - r * 2.0 ** -12)], 1)[None]
    run(dev, io, torch.ones(1, 1, H, 2), torch.zeros(1, 1, H, 2), torch.zeros(1, 1, H, Dv), torch.zeros(1, 1, H), torch.zeros(1, 1, H), h0)


def orthogonal_tokens(H):
    """Two tokens with keys e_0 and e_1 and values 1 and -1, a third that asks for both."""
    q, k, v = torch.zeros(1, 3, H, 2), torch.zeros(1, 3, H, 2), torch.zeros(1, 3, H, 1)
    q[:, 2] = 1
    k[:, 0, :, 0] = k[:, 1, :, 1] = 1
    v[:, 0], v[:, 1] = 1, -1
    return q, k, v


@pytest.mark.parametrize("io", [BF16, F16])
def test_corrections_that_cancel(dev, io):
    """o = beta_0 - beta_1 with beta = x and x (1 - r 2^-12), in float32."""
    H = 64
    x, r = torch.rand(2, H, generator=torch.Generator().manual_seed(1))
    beta = torch.stack([0.5 + x / 2, (0.5 + x / 2) * (1 - r * 2.0 ** -12), x])[None]
    run(dev, io, *orthogonal_tokens(H), torch.zeros(1, 3, H), beta)


@pytest.mark.parametrize("io", [BF16, F16])
def test_decays_that_cancel(dev, io):
    """o = e^{g_1 + g_2} - e^{g_2} with g_1 = -r 2^-12 and g_2 = -x."""
    H = 64
    x, r = torch.rand(2, H, generator=torch.Generator().manual_seed(2))
    g = torch.stack([0 * x, -r * 2.0 ** -12, -x])[None]
    run(dev, io, *orthogonal_tokens(H), g, torch.ones(1, 3, H))


@pytest.mark.parametrize("scale", [0.0, 1e-60])
@pytest.mark.parametrize("io", [torch.float32, BF16, F16])
def test_a_scale_of_zero(dev, scale, io):
    """No scale (1e-60 is 0 in float32): outputs and dq are 0, through the norm too; the last state's gradients are
    what they are."""
    a, do, dl = make(dev, 2, 70, 1, 2, 40, 24, io, seed=61)
    a = {n: t.requires_grad_() for n, t in a.items()}
    o, last = ssm_scan.gated_delta_rule(**a, scale=scale, qk_norm=True, return_last_state=True)
    grads = dict(zip(a, torch.autograd.grad([o, last], list(a.values()), [do, dl])))
    _, want_last, want = delta_ref.delta(**a, scale=0.0, qk_norm=True, dlast=dl)
    assert not o.any() and not grads["q"].any()
    close("last", last, want_last, io)
    for n in ("k", "v", "g", "beta", "h0"):
        close("d" + n, grads[n], want[n], io, grad=True, size=want["size"].get(n, 0.0))
