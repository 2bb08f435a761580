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


def test_generate_goes_on_where_a_row_has_no_distribution(dev):
    """Such a row gives -1, and the model is never given that as an id."""
    lm = block.MambaLM(n_layers=2, d_model=64).to(dev).eval()
    prompt = torch.randint(0, 256, (3, 12), device=dev)
    seen = []
    lm.register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
    head = lm.head.register_forward_hook(lambda mod, args, out: out.index_fill(0, torch.tensor([1], device=dev), float("nan")))
    out = lm.generate(prompt, 5, top_p=0.9)
    head.remove()
    assert (out[1, 12:] == -1).all() and (out[[0, 2]] >= 0).all()
    assert len(seen) == 5 and all(int(s.min()) >= 0 for s in seen)
