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


def walk_inputs(dev, B, Dv):
    g = torch.Generator(device=dev).manual_seed(52)

    def rn(*s):
        return torch.randn(*s, generator=g, device=dev)

    return dict(q=rn(B, 1, 1, 1), k=rn(B, 1, 1, 1), v=rn(B, 1, 1, Dv), g=-rn(B, 1, 1).abs(), beta=torch.sigmoid(rn(B, 1, 1)))


# 2^20 tiles of 16 columns a head, two to a workgroup of 512 threads: 17 heads are more than 2^32 threads
COLUMNS = [slice(c, c + 40) for c in (0, (1 << 23) - 20, (1 << 24) - 40)]


def test_walk_of_more_workgroups_than_a_grid_row(dev):
    B, Dv = 17, 1 << 24
    a = walk_inputs(dev, B, Dv)
    o, last = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    for c in COLUMNS:
        want_o, want_last = delta_ref.delta(**{**a, "v": a["v"][..., c]}, qk_norm=True)
        close("o", o[..., c], want_o, F32)
        close("last", last[..., c], want_last, F32)


def test_backward_walk_of_more_workgroups_than_a_grid_row(dev):
    """dv's columns hang on their own columns of v and the outputs' gradient alone."""
    if torch.cuda.mem_get_info()[0] < 230e9:
        pytest.skip("keeps 10 KB for each of 2^24 tiles: 180 GB")
    B, Dv = 17, 1 << 24
    a = walk_inputs(dev, B, Dv)
    do = torch.randn(B, 1, 1, Dv, device=dev)
    o = ssm_scan.gated_delta_rule(**{**a, "v": a["v"].requires_grad_()}, qk_norm=True)
    dv = torch.autograd.grad(o, a["v"], do)[0]
    for c in COLUMNS:
        _, _, want = delta_ref.delta(**{**a, "v": a["v"][..., c]}, qk_norm=True, dout=do[..., c])
        close("dv", dv[..., c], want["v"], F32, grad=True)
    del o, dv, do, a
    torch.cuda.empty_cache()   # for the tests that follow


def test_batch_rows_and_heads_far_apart(dev):
    """Rows of the operands, and of the outputs' gradient, 2^31 and more elements apart."""
    B, L, H, D, far = 2, 70, 2, 16, (1 << 31) + 8
    g = torch.Generator(device=dev).manual_seed(53)
    buf = torch.empty(far + 4 * L * H * D, device=dev, dtype=torch.bfloat16)

    def spread(i):   # part i of the buffer
        t = buf.as_strided((B, L, H, D), (far, H * D, D, 1), i * L * H * D)
        return t.copy_(torch.randn(B, L, H, D, generator=g, device=dev))

    q, k, v, do = (spread(i) for i in range(4))
    decay, beta = -torch.rand(B, L, H, generator=g, device=dev), torch.rand(B, L, H, generator=g, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, decay, beta)]
    o = ssm_scan.gated_delta_rule(*leaves, qk_norm=True)
    grads = torch.autograd.grad(o, leaves, do)
    want_o, _, want = delta_ref.delta(*leaves, qk_norm=True, dout=do)
    close("o", o, want_o, torch.bfloat16)
    for n, d in zip(("q", "k", "v", "g", "beta"), grads):
        close("d" + n, d, want[n], torch.bfloat16, grad=True, size=want["size"].get(n, 0.0))
