"""Grouped norm at sizes where one thread per lane of a group, or 64 per channel, are 2^32 and more: a grid row of
that many wraps without an error.  Tolerances of test_gpu_group_norm."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan
from test_gpu_group_norm import BF16, F32, close

pytestmark = pytest.mark.gpu


def test_rows_of_more_lanes_than_a_grid_row(dev):
    """2^26 groups of 17 bf16 channels take 64 lanes each: rows around 2^31 and 2^32 lanes, and the last."""
    R, groups, n = (1 << 20) + 5, 64, 17
    g = torch.Generator(device=dev).manual_seed(41)
    x = torch.randn(R, groups * n, generator=g, device=dev, dtype=BF16)
    w = 1 + 0.2 * torch.randn(groups * n, generator=g, device=dev)
    y = ssm_scan.group_norm(x, groups, w, activation="silu")
    for r in (0, 1 << 19, (1 << 20) - 5):
        rows = slice(max(r - 5, 0), r + 10)
        close(f"y at row {r}", y[rows], delta_ref.group_norm(x[rows], groups, w, activation="silu"))


def test_weight_gradients_of_more_channels_than_a_grid_row(dev):
    """2^26 channels: 64 threads for each of their sums are 2^32."""
    n = 256
    groups = (1 << 18) + 3
    g = torch.Generator(device=dev).manual_seed(42)
    x, dy = (torch.randn(2, groups * n, generator=g, device=dev) for _ in range(2))
    w = (1 + 0.2 * torch.randn(groups * n, generator=g, device=dev)).requires_grad_()
    b = torch.zeros(groups * n, device=dev).requires_grad_()
    y = ssm_scan.group_norm(x, groups, w, b)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    for first in (0, (1 << 17) - 2, groups - 5):
        c = slice(first * n, (first + 5) * n)
        want_y, want = delta_ref.group_norm(x[:, c], 5, w[c], b[c], dout=dy[:, c])
        close("y", y[:, c], want_y)
        close("dweight", dw[c], want["weight"])
        close("dbias", db[c], want["bias"])
