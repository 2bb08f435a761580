"""The draw of the next token at the ends of its settings."""

import pytest
import torch

from oracle import token_ref
import ssm_scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 6, 300, 6000, 40000])
def test_min_p_above_one_keeps_the_first(dev, V):
    """No weight reaches it, so only the first of the order is kept, ties of the largest logit or not."""
    logits = torch.zeros(30, V, device=dev)
    logits[:, V // 2:] = 1.0      # ties from V // 2 on
    u = torch.linspace(0, 0.999, 30, device=dev)
    for kw in (dict(min_p=1.5), dict(min_p=float("inf")), dict(min_p=2.0, top_k=7, top_p=0.9), dict(min_p=torch.full((30,), 1.0001, device=dev))):
        token, lp = ssm_scan.sample(logits, u, **kw)
        assert (token == V // 2).all() and (lp == 0).all(), kw
        want, _ = token_ref.sample(logits, u, **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
        assert token.cpu().tolist() == want.tolist()
    token, _ = ssm_scan.sample(logits, u, min_p=1.0)       # the ties have just that weight
    want, _ = token_ref.sample(logits, u, min_p=1.0)
    assert token.cpu().tolist() == want.tolist() and (V < 6 or token.unique().numel() > 1)
    mixed = torch.tensor([0.5, 3.0], device=dev).repeat(15)
    token, _ = ssm_scan.sample(logits, u, min_p=mixed)
    assert (token[1::2] == V // 2).all()


@pytest.mark.parametrize("V", [1 << 22, 1 << 24])
def test_the_largest_vocabularies(dev, V):
    """What is kept of a long row is drawn as from a row of the kept alone."""
    logits = torch.randn(2, V, device=dev, generator=torch.Generator(dev).manual_seed(V))
    u = torch.tensor([0.37, 0.91], device=dev)
    top, at = torch.topk(logits, 50)
    at = at.sort(-1).values
    for kw in (dict(top_k=50), dict(top_k=50, top_p=0.7, temperature=1.3), dict(top_k=50, min_p=0.5)):
        token, lp = ssm_scan.sample(logits, u, **kw)
        want, wp = token_ref.sample(logits.gather(-1, at), u, **kw)
        assert token.tolist() == at.cpu().gather(-1, torch.from_numpy(want)[:, None])[:, 0].tolist()
        # weights of 2^-S steps, S = 37 at 2^24: 50 of them off by half a step each
        assert (lp.double().cpu() - torch.from_numpy(wp)).abs().max() <= 2.0 ** -23 * 8 + 50 * 2.0 ** -37


def test_settings_that_are_no_numbers(dev):
    logits, u = torch.zeros(2, 10, device=dev), torch.rand(2, device=dev)
    for kw in (dict(temperature=None), dict(temperature="1"), dict(top_k=2.5), dict(top_k="3"), dict(top_p="x"), dict(min_p=[0.1, 0.2])):
        with pytest.raises(TypeError, match=next(iter(kw))):
            ssm_scan.sample(logits, u, **kw)
