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


def test_a_second_derivative_is_refused(dev):
    """First gradients are the same under create_graph; differentiating them raises, by every way to the leaves."""
    a, do, dl = make(dev, 1, 70, 1, 2, 16, 8, F32)
    leaves = [t.requires_grad_() for t in a.values()] + [do.requires_grad_()]

    def grads(create_graph):
        o, last = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
        return torch.autograd.grad([o, last], list(a.values()), [do, dl], create_graph=create_graph)

    once, graph = grads(False), grads(True)
    assert all(torch.equal(x, y) and not x.requires_grad and y.requires_grad for x, y in zip(once, graph))
    for g in graph:
        for leaf in leaves:
            with pytest.raises(RuntimeError, match="twice"):
                torch.autograd.grad(g.sum() + 0 * leaf.sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward(retain_graph=True)


def test_a_second_derivative_through_casts_is_refused(dev):
    """Operands that the kernels read as copies."""
    a, do, _ = make(dev, 1, 20, 1, 2, 16, 8, BF16)
    a["v"], a["g"] = a["v"].float().requires_grad_(), a["g"].double().requires_grad_()
    o = ssm_scan.gated_delta_rule(**a)
    dv, dg = torch.autograd.grad(o, [a["v"], a["g"]], do.float(), create_graph=True)
    for d in (dv, dg):
        for leaf in (a["v"], a["g"]):
            with pytest.raises(RuntimeError, match="twice"):
                torch.autograd.grad(d.sum(), leaf, retain_graph=True)


def test_a_second_derivative_of_the_norm_is_refused(dev):
    x, w, b, gate = (torch.randn(s, device=dev).requires_grad_() for s in ((3, 8), (8,), (8,), (3, 8)))
    dy = torch.randn(3, 8, device=dev).requires_grad_()
    leaves = [x, w, b, gate]

    def grads(create_graph):
        return torch.autograd.grad(ssm_scan.group_norm(x, 2, w, b, gate=gate), leaves, dy, create_graph=create_graph)

    once, graph = grads(False), grads(True)
    assert all(torch.equal(p, q) and not p.requires_grad and q.requires_grad for p, q in zip(once, graph))
    for g in graph:
        for leaf in leaves + [dy]:
            with pytest.raises(RuntimeError, match="twice"):
                torch.autograd.grad(g.sum(), leaf, retain_graph=True)
    # only the weight's: the others have no gradient at all
    d = torch.autograd.grad(ssm_scan.group_norm(x.detach(), 2, w), w, dy.detach(), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(d.sum(), w)


@pytest.mark.parametrize("name", ["h0", "q", "k", "v", "g", "beta"])
def test_a_step_that_would_lose_a_gradient_is_refused(dev, name):
    a, _, _ = make(dev, 2, 1, 1, 2, 16, 8, F32)
    one = {n: t if n == "h0" else t[:, 0] for n, t in a.items()}
    h, ops = one["h0"].clone(), ("q", "k", "v", "g", "beta")
    want = ssm_scan.gated_delta_step(h, *(one[n] for n in ops))
    one[name] = one[name].detach().requires_grad_()
    before = one["h0"].detach().clone()
    with pytest.raises(RuntimeError, match="not differentiable"):
        ssm_scan.gated_delta_step(one["h0"], *(one[n] for n in ops))
    assert torch.equal(one["h0"], before)
    with torch.no_grad():
        assert torch.equal(ssm_scan.gated_delta_step(one["h0"], *(one[n] for n in ops)), want)
    assert torch.equal(one["h0"].detach(), h)


def test_a_step_counts_as_a_change_of_its_state(dev):
    """A graph that has kept the state finds it changed, as after any operation in place."""
    a, _, _ = make(dev, 2, 1, 1, 2, 16, 8, F32)
    w = torch.ones_like(a["h0"]).requires_grad_()
    y = (w * a["h0"]).sum()
    ssm_scan.gated_delta_step(a["h0"], *(a[n][:, 0] for n in ("q", "k", "v", "g", "beta")))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        ssm_scan.gated_delta_step(torch.zeros_like(a["h0"]), *(a[n][:, 0] for n in ("q", "k", "v", "g", "beta")))


@pytest.mark.parametrize("empty", ["B", "L"])
def test_no_tokens_give_new_tensors_in_the_graph(dev, empty):
    """No batch rows or no tokens: o and last are new tensors, and every operand has its (empty or passed on) gradient."""
    a, _, _ = make(dev, 2, 3, 1, 2, 16, 8, F32)
    a = {n: (t[:0] if empty == "B" else t if n == "h0" else t[:, :0]).detach().requires_grad_() for n, t in a.items()}
    o, last = ssm_scan.gated_delta_rule(**a, return_last_state=True)
    assert torch.equal(last, a["h0"]) and last.data_ptr() != a["h0"].data_ptr() or not last.numel()
    assert o.dtype == a["v"].dtype and o.shape == a["v"].shape
    grads = torch.autograd.grad([o, last], list(a.values()), [torch.ones_like(o), torch.full_like(last, 3.0)])
    for n, d in zip(a, grads):
        assert d.shape == a[n].shape and d.dtype == a[n].dtype and bool((d == 3).all())
    with torch.no_grad():
        last = ssm_scan.gated_delta_rule(**a, return_last_state=True)[1]
        last.zero_()
    assert a["h0"].any() or not a["h0"].numel()


def test_no_streams_to_step(dev):
    a, _, _ = make(dev, 2, 1, 1, 2, 16, 8, BF16)
    o = ssm_scan.gated_delta_step(a["h0"][:0], *(a[n][:0, 0] for n in ("q", "k", "v", "g", "beta")))
    assert o.shape == (0, 2, 8) and o.dtype == BF16
    with pytest.raises(ValueError):   # checked all the same
        ssm_scan.gated_delta_step(a["h0"][:0], *(a[n][:0, 0] for n in ("q", "k", "v", "g")), a["beta"][:1, 0])


def test_a_norm_of_no_rows_is_checked_and_in_the_graph(dev):
    x, gate = (torch.zeros(0, 5, 32, device=dev, dtype=BF16).requires_grad_() for _ in range(2))
    w, b = (torch.ones(32, device=dev).requires_grad_() for _ in range(2))
    y = ssm_scan.group_norm(x, 4, w, b, gate=gate)
    assert y.shape == x.shape and y.dtype == BF16
    for t, d in zip((x, w, b, gate), torch.autograd.grad(y, (x, w, b, gate), torch.ones_like(y))):
        assert d.shape == t.shape and d.dtype == t.dtype and not d.any()
    for kw in (dict(groups=5), dict(groups=0), dict(groups=4, weight=w[:8]), dict(groups=4, gate=gate[:, :2])):
        with pytest.raises(ValueError):
            ssm_scan.group_norm(x, **kw)
    with pytest.raises(TypeError):
        ssm_scan.group_norm(x.double(), 4)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
@pytest.mark.parametrize("name", ["weight", "bias", "gate"])
def test_a_norm_over_two_devices_is_refused(dev, name):
    a = dict(weight=torch.ones(8, device=dev), bias=torch.ones(8, device=dev), gate=torch.ones(3, 8, device=dev))
    a[name] = a[name].to("cuda:1")
    with pytest.raises(ValueError, match="tensors on"):
        ssm_scan.group_norm(torch.ones(3, 8, device=dev), 2, **a)
