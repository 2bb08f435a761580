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


def test_results_change_in_place(dev):
    x, w, r = leaf(dev, 3, 5, 16), leaf(dev, 8, 16, seed=1), leaf(dev, 3, 5, 8, seed=2)
    dy = torch.randn(3, 5, 8, device=dev).to(BF16)
    want = torch.autograd.grad(ssm_scan.linear_act(x, w, activation="gelu", residual=r), [x, w, r], dy)
    y = ssm_scan.linear_act(x, w, activation="gelu", residual=r)
    y.mul_(2)
    y += 1
    for a, b in zip(torch.autograd.grad(y, [x, w, r], dy / 2), want):
        assert torch.equal(a, b)
    x, r, w = leaf(dev, 3, 5, 16), leaf(dev, 3, 5, 16, seed=1), leaf(dev, 16, dtype=F32, seed=2)
    dy = torch.randn(3, 5, 16, device=dev).to(BF16)
    want = torch.autograd.grad(ssm_scan.add_rms_norm(x, r, w)[0], [x, r, w], dy)
    y, s = ssm_scan.add_rms_norm(x, r, w)
    y.mul_(2)
    for a, b in zip(torch.autograd.grad(y, [x, r, w], dy / 2), want):
        assert torch.equal(a, b)
    y, s = ssm_scan.add_rms_norm(x, r, w)
    s.add_(1)   # the backward reads it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)


def test_one_channel_with_any_stride(dev):
    def turned(n, dtype=BF16):   # (n, 1) with strides (1, n)
        return torch.randn(1, n, device=dev).to(dtype).t()

    def flat(t):
        return t.reshape(-1).reshape(-1, 1)

    x, r, dy = turned(5), turned(5), turned(5)
    w = torch.ones(1, device=dev)
    assert x.stride() == (1, 5) and flat(x).stride() == (1, 1)
    got, want = ssm_scan.add_rms_norm(x, r, w), ssm_scan.add_rms_norm(flat(x), flat(r), w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    X = flat(x).detach().requires_grad_()
    a, b = (torch.autograd.grad(ssm_scan.add_rms_norm(X, flat(r), w)[0], X, d)[0] for d in (dy, flat(dy)))
    assert torch.equal(a, b)
    for f in (lambda t: ssm_scan.rms_norm_8bit(t, w), ssm_scan.quantize_rows):
        (q, s), (q2, s2) = f(x), f(flat(x))
        assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)
    tokens = torch.tensor([3, 0, 3, 8, 8], device=dev)
    table = turned(9).requires_grad_()
    out = ssm_scan.embedding(tokens, table, 2.0)
    assert torch.equal(out, ssm_scan.embedding(tokens, flat(table), 2.0))
    a, b = (torch.autograd.grad(ssm_scan.embedding(tokens, table, 2.0), table, d)[0] for d in (dy, flat(dy)))
    assert torch.equal(a, b)
    logits, u = turned(4), torch.rand(4, device=dev)
    assert (ssm_scan.sample(logits, u)[0] == 0).all()
    assert torch.equal(ssm_scan.group_norm(x, 1, w), ssm_scan.group_norm(flat(x), 1, w))


def test_calls_without_rows_are_checked(dev):
    x, w = torch.zeros(0, 32, device=dev), torch.ones(32, device=dev)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            ssm_scan.add_rms_norm(x, x, w, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            ssm_scan.rms_norm_8bit(x, w, eps=eps)
    wide = torch.zeros(0, 16385, device=dev)
    with pytest.raises(ValueError, match="16384"):
        ssm_scan.add_rms_norm(wide, wide, wide.new_ones(16385))
    with pytest.raises(ValueError, match="16384"):
        ssm_scan.quantize_rows(wide)
    with pytest.raises(ValueError, match="scale"):
        ssm_scan.embedding(torch.zeros(0, dtype=torch.long, device=dev), torch.zeros(4, 8, device=dev), scale=float("nan"))
    assert ssm_scan.embedding(torch.zeros(0, dtype=torch.long, device=dev), torch.zeros(0, 8, device=dev)).shape == (0, 8)


def test_a_scale_beyond_float32_is_refused(dev):
    t, w = torch.zeros(3, dtype=torch.long, device=dev), torch.zeros(4, 8, device=dev)
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="scale"):
            ssm_scan.embedding(t, w, scale=scale)
    assert not ssm_scan.embedding(t, w, scale=3e38).any()
