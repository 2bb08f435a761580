"""GatedDeltaMixer with a state is inference, whatever the grad mode: outputs and states without a graph."""

import pytest
import torch

from ssm_scan.delta_mixer import GatedDeltaMixer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pieces", [(5, 1, 3), (1, 1), (7,)])
def test_no_graph_with_a_state(dev, pieces):
    torch.manual_seed(0)
    m = GatedDeltaMixer(d_model=64, heads=4, key_dim=16, value_dim=24, key_heads=2).to(dev)
    u = torch.randn(2, sum(pieces), 64, device=dev, requires_grad=True)
    with torch.no_grad():
        want = m(u)
    state, outs, t = m.init_state(2, dev), [], 0
    for n in pieces:
        outs.append(m(u[:, t:t + n], state))
        t += n
        assert not outs[-1].requires_grad and not state.delta.requires_grad and not state.conv.requires_grad
    # two float32 GEMMs, the conv, the rule and the norm: 2^-15 of the largest output
    assert (torch.cat(outs, 1) - want).abs().max().item() <= 2.0 ** -15 * want.abs().max().item()
    assert torch.is_grad_enabled() and m(u).requires_grad   # without a state it is trained


def test_a_float32_state_under_bf16_autocast(dev):
    """As the Mamba mixer, the layer takes a state kept in another type than its activations.  bf16 roundings of 2^-8
    along a chain of six, in either computation."""
    torch.manual_seed(1)
    m = GatedDeltaMixer(d_model=64, heads=4, key_dim=16, value_dim=24, key_heads=2).to(dev)
    u = torch.randn(2, 9, 64, device=dev)
    state, outs, t = m.init_state(2, dev), [], 0
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        want = m(u)
        for n in (5, 1, 2, 1):
            outs.append(m(u[:, t:t + n], state))
            t += n
    assert state.conv.dtype == torch.float32
    assert (torch.cat(outs, 1) - want).abs().max().item() <= 6 * 2.0 ** -8 * want.abs().max().item()
