"""What the operators around the mixers leave in autograd's graph: the gradients they are given keep their history, their
results can be changed in place, operands of one channel may have any stride, calls without rows are checked like others."""

import pytest
import torch

import ssm_scan

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def leaf(dev, *shape, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev).requires_grad_()


@pytest.mark.parametrize("act", [None, "silu"])
def test_linear_leaves_the_given_gradient_alone(dev, act):
    x, w, r = leaf(dev, 6, 16), leaf(dev, 8, 16, seed=1), leaf(dev, 6, 8, seed=2)
    dy = torch.randn(6, 8, device=dev).to(BF16)
    dx, dr = torch.autograd.grad(ssm_scan.linear_act(x, w, activation=act, residual=r), [x, r], dy, create_graph=True)
    assert not dy.requires_grad and dy.grad_fn is None and torch.equal(dr, dy)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()
    # a gradient with a history: the residual's is linear in it
    a = leaf(dev, 6, 8, seed=3)
    dy = a * 2
    before = dy.grad_fn
    dx, dr = torch.autograd.grad(ssm_scan.linear_act(x, w, activation=act, residual=r), [x, r], dy, create_graph=True)
    assert dy.grad_fn is before
    g, = torch.autograd.grad(dr.sum(), a, retain_graph=True)
    assert torch.equal(g, torch.full_like(g, 2))
    g, = torch.autograd.grad((3 * dy).sum(), a, retain_graph=True)
    assert torch.equal(g, torch.full_like(g, 6))
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()


@pytest.mark.parametrize("io,rt", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_norm_leaves_the_given_gradient_of_the_sum_alone(dev, io, rt):
    x, r, w = leaf(dev, 6, 16, dtype=io), leaf(dev, 6, 16, dtype=rt, seed=1), leaf(dev, 16, dtype=F32, seed=2)
    ds = torch.randn(6, 16, device=dev).to(rt)
    dx, dr, dw = torch.autograd.grad(ssm_scan.add_rms_norm(x, r, w)[1], [x, r, w], ds, create_graph=True)
    assert not ds.requires_grad and ds.grad_fn is None
    assert torch.equal(dx, ds.to(io)) and torch.equal(dr, ds) and not dw.any()
    a = leaf(dev, 6, 16, dtype=rt, seed=3)
    ds = a * 2
    before = ds.grad_fn
    dx, dr = torch.autograd.grad(ssm_scan.add_rms_norm(x, r, w)[1], [x, r], ds, create_graph=True)
    assert ds.grad_fn is before
    g, = torch.autograd.grad(dx.float().sum() + dr.sum(), a)
    assert torch.equal(g, torch.full_like(g, 4))
    # through y there is no second derivative
    y, s = ssm_scan.add_rms_norm(x, r, w)
    dx, = torch.autograd.grad([y, s], [x], [torch.ones_like(y), a * 2], create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()
