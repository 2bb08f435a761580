"""A training pass of the gated delta rule and the grouped norm behind it, captured in a HIP graph: every replay
equals the eager pass bit for bit, with eager work, synchronizations and new inputs between the replays.  No eager
graph of the leaves lives while the pass is captured (its nodes belong to another stream)."""

import pytest
import torch

import ssm_scan
from test_gpu_delta import BF16, F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io,shape", [(F32, (2, 150, 1, 2, 64, 48)), (BF16, (9, 100, 4, 8, 128, 64))])
def test_replays_equal_the_eager_pass(dev, io, shape):
    B, L, Hk, H, Dk, Dv = shape
    inputs = [make(dev, *shape, io, seed=s)[0] for s in (81, 82, 83)]
    g = torch.Generator(device=dev).manual_seed(84)
    gate, dy = (torch.randn(B, L, H * Dv, generator=g, device=dev).to(io) for _ in range(2))
    w = torch.ones(H * Dv, device=dev).requires_grad_()
    leaves = {n: t.clone().requires_grad_() for n, t in inputs[0].items()}

    def step():
        o, last = ssm_scan.gated_delta_rule(**leaves, qk_norm=True, return_last_state=True)
        y = ssm_scan.group_norm(o.flatten(-2), H, w, gate=gate, center=False)
        out = torch.autograd.grad([y, last], list(leaves.values()) + [w], [dy, last.detach()])
        return [y.detach(), last.detach()] + list(out)

    def load(a):
        with torch.no_grad():
            for n, t in leaves.items():
                t.copy_(a[n])

    def eager(a):
        load(a)
        out = [t.clone() for t in step()]
        torch.cuda.synchronize()
        return out

    want = [eager(a) for a in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    torch.cuda.synchronize()
    for rep in range(2):
        for a, ref in zip(inputs, want):
            load(a)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, ref)), rep
            assert all(torch.equal(x, y) for x, y in zip(eager(a), ref))
