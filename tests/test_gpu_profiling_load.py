"""GPU: a KernelTimer entered before the binding is loaded records the launches that follow."""

import pytest
import torch

import ssm_scan
from ssm_scan import _abi

pytestmark = pytest.mark.gpu


def test_launches_after_a_late_load_are_timed(dev, monkeypatch):
    x = torch.randn(4, 32, device=dev)
    monkeypatch.setattr(_abi, "_host", None)
    with ssm_scan.KernelTimer() as t:
        ssm_scan.group_norm(x, 4)
    ssm_scan.group_norm(x, 4)
    assert list(t.records) == ["ssm_gnorm_fwd"] and len(t.records["ssm_gnorm_fwd"]) == 1
