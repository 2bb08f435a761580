"""The norm with the residual's addition and its 8-bit rows against the float64 oracle (oracle/token_ref.py).

Tolerances.  A row's sum of squares has at most 32 terms a lane and ten more additions, so r is off by 21 roundings of
float32, y by 25: 25 2^-24 < 2^-19 of the value, before half a step of its type.  The gradient of s has the same sums in
both terms: 2^-18 of the row's largest magnitude.  The weight's gradient adds a slot's rows in float32, at most
R / 1024 + 4 of them, then float64: that many roundings and 25 of the terms' magnitudes."""

import pytest
import torch

from oracle import token_ref
import ssm_scan

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TINY = {t: torch.finfo(t).tiny for t in (F32, BF16, F16)}


def near(name, got, want, abs_tol):
    half, dtype = torch.finfo(got.dtype).eps / 2, got.dtype
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    # below the smallest normal number a step is that number's, so half a step is half * tiny (2^-25 in float16)
    tol = half * want.abs().clamp(min=TINY[dtype]) + torch.as_tensor(abs_tol, dtype=torch.float64)
    assert ((got - want).abs() <= tol).all(), f"{name}: worst {((got - want).abs() / tol).max().item():.3g} x"


def make(dev, shape, io, rt, seed=0):
    r = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=r)

    return (rn(*shape).to(io).to(dev), (2 * rn(*shape)).to(rt).to(dev), (1 + 0.2 * rn(shape[-1])).to(dev), rn(*shape).to(io).to(dev),
            rn(*shape).to(rt).to(dev))


def check(x, res, w, dy, ds):
    leaves = [t.detach().requires_grad_() for t in (x, res, w)]
    y, s = ssm_scan.add_rms_norm(*leaves)
    assert y.dtype == x.dtype and s.dtype == res.dtype and y.shape == s.shape == x.shape
    # the sum of two 16-bit numbers in float32 and its rounding: two roundings at most
    near("s", s, x.double().cpu() + res.double().cpu(), 2.0 ** -24 * (x.double().cpu() + res.double().cpu()).abs())
    want, d, dw, mag = token_ref.norm(s, w, dy=dy, ds=ds)
    near("y", y, want, 2.0 ** -19 * want.abs())
    outs, douts = ([y, s], [dy, ds]) if ds is not None else ([y], [dy])
    dx, dr, dweight = torch.autograd.grad(outs, leaves, douts)
    assert dx.dtype == x.dtype and dr.dtype == res.dtype and dweight.dtype == w.dtype
    top = 2.0 ** -18 * d.abs().amax(-1, keepdim=True)
    near("dx", dx, d, top)
    near("dresidual", dr, d, top)
    rows = x.numel() // x.shape[-1]
    near("dweight", dweight, dw, (rows / 1024 + 29) * 2.0 ** -24 * mag)


PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]


# one row and channel, rows that fill no load, every count of wavefronts and loads a lane, the widest rows, many rows
@pytest.mark.parametrize("io,rt", PAIRS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 3, 33), (5, 64), (9, 250), (4, 512), (3, 1000), (2, 1001), (7, 2048), (1030, 520),
                                   (3, 4096), (2, 5120), (3, 8192), (2, 16384), (1, 16383), (5000, 256), (1500, 1032), (4100, 24)])
def test_sizes(dev, io, rt, shape):
    check(*make(dev, shape, io, rt, seed=len(shape) + shape[-1]))


@pytest.mark.parametrize("io,rt", PAIRS)
def test_sum_or_norm_alone(dev, io, rt):
    x, res, w, dy, ds = make(dev, (40, 384), io, rt, seed=1)
    check(x, res, w, dy, None)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    _, s = ssm_scan.add_rms_norm(*leaves)
    dx, dr, dw = torch.autograd.grad(s, leaves, ds)
    assert torch.equal(dx, ds.to(io)) and torch.equal(dr, ds) and not dw.any()


def test_strided_rows_and_frozen_operands(dev):
    x, res, w, dy, ds = make(dev, (30, 256), BF16, BF16, seed=2)
    y, s = ssm_scan.add_rms_norm(x, res, w)
    both = torch.cat([x, res], -1)
    y2, s2 = ssm_scan.add_rms_norm(both[:, :256], both[:, 256:], w)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    odd = torch.cat([x[:, :3], x, res], -1)   # rows at no whole load
    y3, s3 = ssm_scan.add_rms_norm(odd[:, 3:259], odd[:, 259:], w)
    assert torch.equal(s, s3)
    near("y", y3, token_ref.norm(s, w), 2.0 ** -19 * y.double().cpu().abs())
    y4, s4 = ssm_scan.add_rms_norm(torch.stack([x, x], -1)[..., 0], res, w.double())
    assert torch.equal(y, y4) and torch.equal(s, s4)
    for which in range(3):
        leaves = [x.detach(), res.detach(), w.detach()]
        leaves[which].requires_grad_()
        g, = torch.autograd.grad(list(ssm_scan.add_rms_norm(*leaves)), [leaves[which]], [dy, ds])
        full = [t.detach().requires_grad_() for t in leaves]
        assert torch.equal(g, torch.autograd.grad(list(ssm_scan.add_rms_norm(*full)), full, [dy, ds])[which])
        leaves[which].requires_grad_(False)


def test_zero_rows_and_not_finite_ones(dev):
    """A row of zeros is normalized to zeros; an infinity or NaN stays in its row."""
    x, res, w, dy, ds = make(dev, (8, 128), F32, F32, seed=3)
    x[2] = 0
    res[2] = 0
    check(x, res, w, dy, ds)
    x[5, 7] = float("nan")
    x[6, 9] = float("inf")
    y, s = ssm_scan.add_rms_norm(x, res, w)
    fine = torch.tensor([0, 1, 2, 3, 4, 7], device=dev)
    assert torch.isfinite(y[fine]).all() and torch.isnan(y[5]).all() and torch.isnan(y[6, 9]) and torch.isinf(s[6, 9])


def test_repeatable(dev):
    x, res, w, dy, ds = make(dev, (3000, 512), BF16, BF16, seed=4)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    a = torch.autograd.grad(list(ssm_scan.add_rms_norm(*leaves)), leaves, [dy, ds])
    b = torch.autograd.grad(list(ssm_scan.add_rms_norm(*leaves)), leaves, [dy, ds])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---------------------------------------------------------------- 8-bit rows
def check8(q, scale, y):
    """y in float64: the scale is off by y's 25 roundings and two more; q by half a step of e4m3 (2^-4 of a normal
    value, 2^-10 below 2^-6) of y / scale, itself off by 29 roundings."""
    want = token_ref.rows8_scale(y)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == F32 and q.shape == y.shape and scale.shape == y.shape[:-1]
    assert ((scale.double().cpu() - want).abs() <= 2.0 ** -19 * want).all()
    v = y / scale.double().cpu()[..., None]
    off = (q.float().double().cpu() - v).abs()
    assert (off <= torch.clamp(2.0 ** -4 * v.abs(), min=2.0 ** -10) * (1 + 2.0 ** -18) + 2.0 ** -18 * v.abs()).all()


@pytest.mark.parametrize("io,rt", PAIRS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 36), (64, 512), (5, 1001), (3, 4096), (2, 8192), (1, 16384), (1200, 264)])
def test_8bit_rows(dev, io, rt, shape):
    x, res, w, _, _ = make(dev, shape, io, rt, seed=5)
    q, scale, s = ssm_scan.rms_norm_8bit(x, w, residual=res)
    assert torch.equal(s, ssm_scan.add_rms_norm(x, res, w)[1])
    check8(q, scale, token_ref.norm(s, w))
    q, scale = ssm_scan.rms_norm_8bit(x, w)
    check8(q, scale, token_ref.norm(x, w))
    q, scale = ssm_scan.quantize_rows(x)
    check8(q, scale, x.double().cpu())


def test_8bit_edges(dev):
    x = torch.zeros(7, 24, device=dev)
    x[1, 3] = 1e-45             # the scale is kept from leaving the normal numbers
    x[2, :] = 448.0
    x[3, 5], x[3, 6] = float("nan"), -2.0
    x[4, 5], x[4, 6] = float("inf"), 3.0
    x[5] = -3e38
    x[6, 0] = 1e-30
    q, scale = ssm_scan.quantize_rows(x)
    f = q.float()
    assert scale[0] == 1 and not f[0].any()
    assert scale[1] > 0 and torch.isfinite(f[1]).all()
    assert scale[2] == 1 and (f[2] == 448).all()
    assert torch.isnan(f[3, 5]) and f[3, 6] == -448 and scale[3] == torch.tensor(2.0, device=dev) / 448 and not f[3, :5].any()
    assert torch.isinf(scale[4]) and torch.isnan(f[4, 5]) and f[4, 6] == 0
    assert (f[5] == -448).all() and torch.isfinite(scale[5])
    assert f[6, 0] == 448 and not f[6, 1:].any()


def test_all_8bit_values(dev):
    """Every e4m3 value and every midpoint between two neighbours (to the even one), through a row whose scale is 1."""
    every = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[torch.isfinite(every)]
    pos = torch.unique(every[every >= 0])
    mid = (pos[1:] + pos[:-1]) / 2
    x = torch.cat([every, mid, -mid, torch.tensor([448.0])]).to(dev)[None]
    q, scale = ssm_scan.quantize_rows(x)
    assert scale.item() == 1
    assert torch.equal(q.float().cpu(), x.cpu().to(torch.float8_e4m3fn).float())


def test_refusals_and_no_rows(dev):
    x, w = torch.zeros(4, 32, device=dev), torch.ones(32, device=dev)
    for bad in (dict(residual=x[:2]), dict(weight=w[:8]), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            ssm_scan.add_rms_norm(**{**dict(x=x, residual=x, weight=w), **bad})
    with pytest.raises(ValueError, match="16384"):
        ssm_scan.add_rms_norm(torch.zeros(2, 16385, device=dev), torch.zeros(2, 16385, device=dev), torch.ones(16385, device=dev))
    with pytest.raises(TypeError):
        ssm_scan.add_rms_norm(x.double(), x.double(), w)
    with pytest.raises(TypeError, match="residual"):
        ssm_scan.add_rms_norm(x, x.bfloat16(), w)
    with pytest.raises(TypeError, match="residual"):
        ssm_scan.add_rms_norm(x.bfloat16(), x.half(), w)
    for call in (lambda t: ssm_scan.rms_norm_8bit(t, w), lambda t: ssm_scan.quantize_rows(t), lambda t: ssm_scan.rms_norm_8bit(x, w, residual=t)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_())
    e = x[:0].clone().requires_grad_()
    y, s = ssm_scan.add_rms_norm(e, x[:0], w)
    assert y.shape == s.shape == (0, 32) and y.requires_grad
    q, scale, s = ssm_scan.rms_norm_8bit(x[:0], w, residual=x[:0])
    assert q.shape == (0, 32) and scale.shape == (0,) and s.shape == (0, 32)
    leaf = x.clone().requires_grad_()
    y, _ = ssm_scan.add_rms_norm(leaf, x, w)
    g, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
