"""What the gated delta rule, its step and the grouped norm do not differentiate is refused, never left out."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import ssm_scan
from test_gpu_delta import BF16, F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "h0"])
@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_is_refused(dev, name, reverse):
    a, _, _ = make(dev, 1, 5, 1, 2, 16, 8, F32)
    if reverse:
        a["v" if name != "v" else "q"].requires_grad_()
    with fwd.dual_level():
        a[name] = fwd.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ssm_scan.gated_delta_rule(**a)
        if not reverse:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ssm_scan.gated_delta_step(a["h0"], *(a[n][:, 0] for n in ("q", "k", "v", "g", "beta")))


@pytest.mark.parametrize("name", ["x", "weight", "bias", "gate"])
def test_forward_mode_of_the_norm_is_refused(dev, name):
    a = dict(x=torch.ones(3, 8, device=dev), weight=torch.ones(8, device=dev), bias=torch.ones(8, device=dev),
             gate=torch.ones(3, 8, device=dev))
    with fwd.dual_level():
        a[name] = fwd.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ssm_scan.group_norm(groups=2, **a)
