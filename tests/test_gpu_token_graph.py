"""A captured training pass through the embedding, the residual norm and linear layers of every kind of launch (few rows, split
sums, copied operands, large tiles): two graphs of it, replayed in turn with eager work between, give the eager results."""

import pytest
import torch

import ssm_scan

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("n,D,H", [(20, 256, 1000), (130, 1024, 264), (500, 520, 777), (4096, 256, 3584)])
def test_training_pass_in_two_graphs(dev, n, D, H):
    torch.manual_seed(n)

    def rn(*s):
        return (torch.randn(*s, device=dev) / s[-1] ** 0.5).to(BF16)

    tokens = [torch.randint(-1, 301, (n,), device=dev) for _ in range(2)]
    E, A, B, bias = rn(300, D).requires_grad_(), rn(H, D).requires_grad_(), rn(D, H).requires_grad_(), rn(H).requires_grad_()
    w = torch.ones(D, device=dev, requires_grad=True)
    dout = [rn(n, D), rn(n, D)]
    leaves = [E, A, B, bias, w]

    def step(i):
        x = ssm_scan.embedding(tokens[i], E, scale=16.0)
        y, s = ssm_scan.add_rms_norm(x, x, w)
        h = ssm_scan.linear_act(y, A, bias, "gelu" if i else "silu")
        out = ssm_scan.linear_act(h, B, residual=s)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout[i])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(step(i))
        graphs.append(g)
    for k in range(3):
        for t in tokens:
            t.copy_(torch.roll(t, 7 * k + 1))
        with torch.no_grad():
            A.mul_(1.0 + 0.25 * k)
        want = [step(i) for i in range(2)]
        for g in graphs if k % 2 else graphs[::-1]:
            g.replay()
        junk = torch.full((1 << 20,), float("nan"), device=dev)   # eager work that reuses the eager pool
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(results[i], want[i])), (k, i)
        del junk
