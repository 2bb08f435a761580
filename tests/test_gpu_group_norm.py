"""Grouped norm kernels against the float64 oracle (oracle/delta_ref.py).

Tolerances: half a step of the output's type relative to the value, plus the float32 arithmetic's error:
sums of up to 1024 terms and about ten roundings, 2^-20 of the tensor's largest magnitude (the weights'
gradients, float64 sums of float32 terms over the rows, likewise)."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def close(name, got, want):
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    tol = half * want.abs() + 2.0 ** -20 * want.abs().max()
    assert ((got - want).abs() <= tol).all(), f"{name}: worst {((got - want).abs() / tol).max().item():.3g} x"


def check(x, groups, weight, bias, gate, activation, center, dy):
    leaves = {n: t for n, t in dict(x=x, weight=weight, bias=bias, gate=gate).items() if t is not None}
    for t in leaves.values():
        t.requires_grad_()
    y = ssm_scan.group_norm(x, groups, weight, bias, gate=gate, activation=activation, center=center)
    assert y.dtype == x.dtype and y.shape == x.shape
    want_y, want = delta_ref.group_norm(x, groups, weight, bias, gate, activation, center, dout=dy)
    close("y", y, want_y)
    for n, d in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        assert d.dtype == leaves[n].dtype
        close("d" + n, d, want[n])


def make(dev, shape, io, seed=0):
    r = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=r)

    C = shape[-1]
    return ((rn(*shape) + 0.3 * rn(C)).to(io).to(dev), (1 + 0.2 * rn(C)).to(dev), (0.2 * rn(C)).to(dev), rn(*shape).to(io).to(dev),
            rn(*shape).to(io).to(dev))


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("mode", ["gate", "silu", None])
@pytest.mark.parametrize("center", [False, True])
def test_modes(dev, io, mode, center):
    x, w, b, gate, dy = make(dev, (3, 50, 512), io)
    check(x, 8, w, b, gate if mode == "gate" else None, "silu" if mode == "silu" else None, center, dy)


# one row, one channel per group, groups that fill no lane, the widest group, more rows than row slots
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", [((1, 64), 1), ((7, 6), 6), ((5, 3, 480), 6), ((9, 100), 2), ((4, 1024), 1), ((11, 2000), 2),
                                          ((3, 2048), 16), ((2, 33), 1), ((6000, 24), 3), ((40, 4096), 4), ((5, 510), 2)])
def test_sizes(dev, io, shape, groups):
    x, w, b, gate, dy = make(dev, shape, io, seed=1)
    check(x, groups, w, b, gate, None, True, dy)


def test_without_weights(dev):
    x, _, _, gate, dy = make(dev, (30, 128), F32, seed=2)
    check(x, 4, None, None, gate, None, False, dy)
    x, w, b, _, dy = make(dev, (30, 128), F32, seed=3)
    check(x, 4, w, None, None, None, True, dy)
    x, w, b, _, dy = make(dev, (30, 128), F32, seed=4)
    check(x, 4, None, b, None, "silu", True, dy)


def test_strided_rows_other_types_and_frozen_weights(dev):
    """x and the gate halves of one projection (read in place), at an odd offset too; bf16 weights."""
    x, w, b, gate, dy = make(dev, (20, 256), BF16, seed=5)
    both = torch.cat([x, gate], -1)
    y = ssm_scan.group_norm(both[:, :256], 4, w, b, gate=both[:, 256:])
    assert torch.equal(y, ssm_scan.group_norm(x, 4, w, b, gate=gate))
    odd = torch.cat([x[:, :3], x, gate], -1)
    close("y", ssm_scan.group_norm(odd[:, 3:259], 4, w, b, gate=odd[:, 259:]), delta_ref.group_norm(x, 4, w, b, gate))
    t = torch.stack([x, x], -1)[..., 0]
    assert torch.equal(y, ssm_scan.group_norm(t, 4, w, b, gate=gate))
    check(x, 4, w.bfloat16(), b.bfloat16(), gate, None, True, dy)
    x2 = x.detach().requires_grad_()
    ssm_scan.group_norm(x2, 4, w.detach(), gate=gate.detach()).backward(dy)   # only x needs a gradient
    close("dx", x2.grad, delta_ref.group_norm(x, 4, w, None, gate, dout=dy)[1]["x"])


def test_constant_rows_and_repeatable_backward(dev):
    """A row of one value has no variance: y is the bias, and the gradients stay finite."""
    x, w, b, _, dy = make(dev, (600, 128), F32, seed=6)
    x[3] = 5.0
    x[4] = 0.0
    check(x, 4, w, b, None, None, True, dy)
    y = ssm_scan.group_norm(x, 4, w, b)
    a1 = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
    a2 = torch.autograd.grad(y, [x, w, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(a1, a2))


def test_refusals_and_no_rows(dev):
    x = torch.zeros(4, 32, device=dev)
    for kw in (dict(groups=5), dict(groups=0), dict(groups=4, weight=x[0, :8]), dict(groups=4, gate=x[:2]), dict(groups=4, eps=-1.0)):
        with pytest.raises(ValueError):
            ssm_scan.group_norm(x, **kw)
    with pytest.raises(ValueError, match="group_size"):
        ssm_scan.group_norm(torch.zeros(2, 1025, device=dev), 1)
    with pytest.raises(TypeError):
        ssm_scan.group_norm(x.double(), 4)
    assert ssm_scan.group_norm(x[:0], 4).shape == (0, 32)
