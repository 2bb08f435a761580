"""The operators of the token's path where the package's own models call them: an output projection of another kind, a
model whose logits are no numbers, a float64 model."""

import pytest
import torch
import torch.nn as nn

from ssm_scan import block
from ssm_scan.delta_mixer import GatedDeltaMixer

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def mixer(dev):
    torch.manual_seed(0)
    m = GatedDeltaMixer(64, heads=2, key_dim=32).to(dev)
    for part in (m.in_proj, m.conv, m.out_proj):
        part.to(BF16)
    return m


class Doubled(nn.Linear):
    def forward(self, x):
        return super().forward(x) * 2


def test_other_output_projections_of_the_mixer(dev):
    m = mixer(dev)
    u, r = (torch.randn(2, 9, 64, device=dev).to(BF16) for _ in range(2))
    with torch.no_grad():
        plain = m(u)
        bias = torch.randn(64, device=dev).to(BF16)
        m.out_proj.bias = nn.Parameter(bias)
        got = m(u, residual=r)
        want = plain.float() + bias.float() + r.float()
        # a rounding of plain (2^-9 of it), one of the result
        assert ((got.float() - want).abs() <= 2.0 ** -8 * (plain.float().abs() + want.abs())).all()
        m = mixer(dev)
        h = m.out_proj.register_forward_hook(lambda mod, args, out: out * 2)
        assert torch.equal(m(u, residual=r), r + plain * 2)
        h.remove()
        w = m.out_proj.weight
        m.out_proj = Doubled(m.out_proj.in_features, 64, bias=False).to(dev).to(BF16)
        m.out_proj.weight = w
        assert torch.equal(m(u, residual=r), r + plain * 2)
