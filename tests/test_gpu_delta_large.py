"""The gated delta rule at sizes whose workgroups together have 2^32 threads and more: a grid row of that many
wraps without an error.  Tolerances of test_gpu_delta."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan
from test_gpu_delta import F32, close

pytestmark = pytest.mark.gpu


def test_step_of_more_workgroups_than_a_grid_row(dev):
    """2^24 heads over the streams, a workgroup of 256 threads each: streams around 2^31 and 2^32 threads, and the last."""
    B, H, Dk, Dv = (1 << 21) + 3, 8, 2, 4
    g = torch.Generator(device=dev).manual_seed(51)

    def rn(*s):
        return torch.randn(*s, generator=g, device=dev)

    q, k, v, decay, beta, h = rn(B, H, Dk), rn(B, H, Dk), rn(B, H, Dv), -rn(B, H).abs(), torch.sigmoid(rn(B, H)), rn(B, H, Dk, Dv)
    before = h.clone()
    o = ssm_scan.gated_delta_step(h, q, k, v, decay, beta, qk_norm=True)
    for first in (0, (1 << 20) - 5, B - 10):
        r = slice(first, first + 10)
        want_o, want_h = delta_ref.delta(*(t[r, None] for t in (q, k, v, decay, beta)), h0=before[r], qk_norm=True)
        close("o", o[r], want_o[:, 0], F32)
        close("h", h[r], want_h, F32)
