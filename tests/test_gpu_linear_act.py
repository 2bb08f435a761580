"""The linear layer with its epilogue, in 16 and 8 bits, against the float64 oracle (oracle/token_ref.py).

Tolerances.  Products of 16- and 8-bit numbers are exact in float32.  A sum of K of them passes K / 32 matrix
instructions, each adding its 32 in at most 32 steps, and up to 16 partial sums: (K / 32 + 64) 2^-24 of the terms' magnitudes.
The epilogue adds four roundings; silu and gelu (slope at most 1.13) are formed within 2^-20 of their value and 2^-21 of z.
The backward reads z rounded to 16 bits, half a step of |z| that the second derivative (0.8 at most) brings into dz; dz
is rounded to 16 bits; its products as above.
8 bits: the matrix instructions add 8 products at a time in steps of 2^-13 of the largest one's power of two (found with
one large and seven small products), so each of the other 7 is off by that at most: 7 2^-13 of the terms' magnitudes beside
the above.  Where products differ by less than 2^13 from the smallest's last bit on, as small whole numbers do, nothing is lost."""

import pytest
import torch

from oracle import token_ref
import ssm_scan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def near(name, got, want, tol):
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).tiny
    got, want = got.detach().double().cpu().reshape(want.shape), want
    assert torch.isfinite(got).all(), name
    # below the smallest normal number a step is that number's
    tol = half * want.abs().clamp(min=tiny) + tol
    off = (got - want).abs()
    assert (off <= tol).all(), f"{name}: worst {(off / tol).max().item():.3g} x at {int((off / tol).argmax())}"


def make(dev, shape, N, io, seed=0):
    r = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=r)

    K = shape[-1]
    return (rn(*shape).to(io).to(dev), (rn(N, K) / K ** 0.5).to(io).to(dev), (0.5 * rn(N)).to(io).to(dev),
            rn(*shape[:-1], N).to(io).to(dev), rn(*shape[:-1], N).to(io).to(dev))


def check(x, w, bias, act, res, dy):
    leaves = {n: t.detach().requires_grad_() for n, t in dict(x=x, weight=w, bias=bias, residual=res).items() if t is not None}
    y = ssm_scan.linear_act(leaves["x"], leaves["weight"], leaves.get("bias"), act, leaves.get("residual"))
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    r = token_ref.linear(x, w, bias, act, res, dy)
    K, half = x.shape[-1], torch.finfo(x.dtype).eps / 2
    grow = lambda k: (k / 32 + 64) * 2.0 ** -24
    ztol = grow(K) * r["mag"]
    ytol = 1.13 * ztol + 2.0 ** -20 * (r["y"].reshape(r["z"].shape).abs() + r["z"].abs() + (0 if res is None else r["dresidual"].abs() * 0 + token_ref.wide(res).reshape(r["z"].shape).abs()))
    near("y", y, r["y"].reshape(r["z"].shape), ytol)
    with torch.no_grad():
        assert torch.equal(y, ssm_scan.linear_act(x, w, bias, act, res))
    if dy is None:
        return
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    dz, d = r["dz"], r["dy"].abs()
    dztol = torch.zeros_like(dz)
    if act:   # z as it was kept, and dz as it is stored
        dztol = d * (0.8 * (half * r["z"].abs() + ztol) + 2.0 ** -20) + half * dz.abs() + torch.finfo(x.dtype).tiny
    M = dz.shape[0]
    near("dx", grads["x"], r["dx"], (dztol + grow(dz.shape[1]) * dz.abs()) @ r["w"].abs())
    near("dweight", grads["weight"], r["dw"], (dztol + grow(M) * dz.abs()).t() @ r["x"].abs())
    if bias is not None:   # of dz before it is stored; float32 sums of up to M terms, then float64
        near("dbias", grads["bias"], r["dbias"], (dztol + (M / 64 + 8) * 2.0 ** -24 * dz.abs()).sum(0))
    if res is not None:
        assert torch.equal(grads["residual"], dy)


# ---------------------------------------------------------------- 16 bits
# one of everything; sizes that fill no tile, load or step; sizes of whole tiles; few rows; few columns; a long sum; many tiles
SIZES = [((1, 1), 1), ((3, 5), 7), ((2, 3, 17), 9), ((1, 64), 64), ((16, 128), 48), ((33, 72), 40), ((64, 64), 64), ((128, 256), 256),
         ((100, 515), 333), ((7, 2048), 24), ((1, 4096), 1000), ((257, 40), 300), ((300, 1024), 520), ((512, 512), 768), ((1, 8), 2001),
         ((40, 8200), 16), ((640, 96), 1280), ((5, 32), 1)]


@pytest.mark.parametrize("io", [BF16, F16])
@pytest.mark.parametrize("shape,N", SIZES)
def test_sizes(dev, io, shape, N):
    x, w, bias, res, dy = make(dev, shape, N, io, seed=N)
    check(x, w, bias, "silu", res, dy)


@pytest.mark.parametrize("io", [BF16, F16])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M", [1, 50, 300])
def test_epilogues(dev, io, act, bias, res, M):
    x, w, b, r, dy = make(dev, (M, 264), 136, io, seed=1)
    check(x, w, b if bias else None, act, r if res else None, dy)


def test_strides(dev):
    """Rows of a larger tensor, at any offset, a transposed weight, a broadcast row."""
    x, w, b, r, dy = make(dev, (70, 256), 128, BF16, seed=2)
    ref = ssm_scan.linear_act(x, w, b, "gelu", r)
    wide = torch.cat([x, w[:70, :256]], 1)
    assert torch.equal(ref, ssm_scan.linear_act(wide[:, :256], w, b, "gelu", r))
    for off in (1, 3, 8):
        odd = torch.cat([x[:, :off], x], 1)
        ow = torch.cat([w[:, :off], w], 1)
        orr = torch.cat([r[:, :off], r], 1)
        y = ssm_scan.linear_act(odd[:, off:], ow[:, off:], b, "gelu", orr[:, off:])
        near("y", y, ref.double().cpu(), 2 * torch.finfo(BF16).eps * ref.double().cpu().abs() + 1e-4)
        check(odd[:, off:], ow[:, off:], b, "gelu", orr[:, off:], torch.cat([dy[:, :off], dy], 1)[:, off:])
    check(x.t().contiguous().t(), w.t().contiguous().t(), b, "silu", r.t().contiguous().t(), dy.t().contiguous().t())
    check(x[:1].expand(70, 256), w, torch.stack([b, b], 1)[:, 0], None, r[:, :1].expand(70, 128), dy[:1].expand(70, 128))


def test_frozen_operands(dev):
    x, w, b, r, dy = make(dev, (40, 96), 64, BF16, seed=3)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    full = torch.autograd.grad(ssm_scan.linear_act(*leaves[:3], "silu", leaves[3]), leaves, dy)
    for i in range(4):
        one = [t.detach() for t in (x, w, b, r)]
        one[i].requires_grad_()
        g, = torch.autograd.grad(ssm_scan.linear_act(*one[:3], "silu", one[3]), [one[i]], dy)
        assert torch.equal(g, full[i]), i
        one[i].requires_grad_(False)


def test_not_finite_rows_stay_theirs(dev):
    x, w, b, r, _ = make(dev, (20, 100), 60, BF16, seed=4)
    x[3, 5], x[11, 99] = float("inf"), float("nan")
    y = ssm_scan.linear_act(x, w, b, "silu", r)
    fine = [i for i in range(20) if i not in (3, 11)]
    assert torch.isfinite(y[fine]).all() and torch.isnan(y[11]).all() and not torch.isfinite(y[3]).all()
    w[7, 3] = float("nan")
    y = ssm_scan.linear_act(x[:3], w, b, "silu", r[:3])
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, :7]).all() and torch.isfinite(y[:, 8:]).all()


def test_repeatable(dev):
    x, w, b, r, dy = make(dev, (33, 4096), 200, BF16, seed=5)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def step():
        y = ssm_scan.linear_act(*leaves[:3], "silu", leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    assert all(torch.equal(p, q) for p, q in zip(step(), step()))


# ---------------------------------------------------------------- 8 bits
@pytest.mark.parametrize("io", [BF16, F16])
@pytest.mark.parametrize("shape,N", SIZES + [((64, 4096), 512), ((3, 130), 130), ((200, 16), 16)])
def test_8bit(dev, io, shape, N):
    x, w, b, r, _ = make(dev, shape, N, io, seed=6)
    (q, s), (wq, ws) = ssm_scan.quantize_rows(x), ssm_scan.quantize_rows(w)
    for act, bias, res in ((None, None, None), ("silu", b, None), ("gelu", b, r)):
        y = ssm_scan.linear_8bit(q, s, wq, ws, bias=bias, activation=act, residual=res, dtype=io)
        assert y.dtype == io and y.shape == shape[:-1] + (N,)
        t = token_ref.linear(q.double().cpu() * s.double().cpu()[..., None], wq.double().cpu() * ws.double().cpu()[:, None], bias, act, res)
        K = shape[-1]
        ztol = ((K / 32 + 64) * 2.0 ** -24 + 7 * 2.0 ** -13) * t["mag"]
        ytol = 1.13 * ztol + 2.0 ** -20 * (t["y"].reshape(ztol.shape).abs() + t["z"].abs() + (0 if res is None else token_ref.wide(res).reshape(ztol.shape).abs()))
        near("y", y, t["y"].reshape(ztol.shape), ytol)


@pytest.mark.parametrize("io", [BF16, F16])
@pytest.mark.parametrize("shape,N", SIZES + [((64, 4096), 512), ((3, 130), 130), ((200, 16), 16), ((700, 1024), 700)])
def test_8bit_whole_numbers(dev, io, shape, N):
    """Products of up to 4 x 4 and sums below 2^24: z is exact, and only the epilogue rounds."""
    r = torch.Generator().manual_seed(8)
    x, w = (torch.randint(-4, 5, s, generator=r).float() for s in (shape, (N, shape[-1])))
    s, ws = torch.rand(shape[:-1], generator=r) + 0.5, (torch.rand(N, generator=r) + 0.5) / shape[-1]
    y = ssm_scan.linear_8bit(x.to(torch.float8_e4m3fn).to(dev), s.to(dev), w.to(torch.float8_e4m3fn).to(dev), ws.to(dev), dtype=io)
    z = (x.double().reshape(-1, shape[-1]) @ w.double().t()) * s.double().reshape(-1, 1) * ws.double()
    near("y", y, z, 3 * 2.0 ** -24 * z.abs())


def test_8bit_strides(dev):
    x, w, b, r, _ = make(dev, (70, 256), 128, BF16, seed=7)
    (q, s), (wq, ws) = ssm_scan.quantize_rows(x), ssm_scan.quantize_rows(w)
    ref = ssm_scan.linear_8bit(q, s, wq, ws, b, "silu", r)
    both = torch.cat([q.view(torch.uint8), wq.view(torch.uint8)[:70]], 1).view(torch.float8_e4m3fn)
    assert torch.equal(ref, ssm_scan.linear_8bit(both[:, :256], s, wq, ws, b, "silu", r))
    odd = torch.cat([q.view(torch.uint8)[:, :3], q.view(torch.uint8)], 1).view(torch.float8_e4m3fn)
    y = ssm_scan.linear_8bit(odd[:, 3:], torch.stack([s, s], 1)[:, 0], wq, ws, b, "silu", r)
    near("y", y, ref.double().cpu(), 2 * torch.finfo(BF16).eps * ref.double().cpu().abs() + 1e-4)


# ---------------------------------------------------------------- refusals
def test_refusals_and_no_rows(dev):
    x, w, b, r, _ = make(dev, (4, 32), 16, BF16)
    for bad, err in ((dict(weight=w[:, :8]), ValueError), (dict(weight=w[0]), ValueError), (dict(bias=b[:3]), ValueError),
                     (dict(residual=r[:2]), ValueError), (dict(activation="tanh"), ValueError), (dict(x=x.float(), weight=w.float()), TypeError),
                     (dict(weight=w.half()), TypeError), (dict(bias=b.float()), TypeError), (dict(residual=r.float()), TypeError),
                     (dict(weight=w[:0]), ValueError)):
        with pytest.raises(err):
            ssm_scan.linear_act(**{**dict(x=x, weight=w, bias=b, residual=r), **bad})
    (q, s), (wq, ws) = ssm_scan.quantize_rows(x), ssm_scan.quantize_rows(w)
    for bad, err in ((dict(q=x), TypeError), (dict(scale=s[:2]), ValueError), (dict(scale=s.half()), TypeError), (dict(weight_scale=s), ValueError),
                     (dict(dtype=torch.float32), TypeError), (dict(bias=b.half()), TypeError), (dict(weight=w), TypeError)):
        with pytest.raises(err):
            ssm_scan.linear_8bit(**{**dict(q=q, scale=s, weight=wq, weight_scale=ws), **bad})
    with pytest.raises(RuntimeError, match="not differentiable"):
        ssm_scan.linear_8bit(q, s, wq, ws, bias=b.clone().requires_grad_())
    e = x[:0].clone().requires_grad_()
    y = ssm_scan.linear_act(e, w, b, "silu", r[:0])
    assert y.shape == (0, 16) and y.requires_grad
    assert ssm_scan.linear_8bit(q[:0], s[:0], wq, ws).shape == (0, 16)
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(ssm_scan.linear_act(leaf, w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_views_that_end_with_their_storage(dev):
    """Rows of whole loads whose last one ends inside a load, at the end of the memory that is theirs."""
    for io in (BF16, F16):
        x, w, b, r, dy = make(dev, (70, 515), 136, io, seed=9)
        sx, sw = torch.zeros(69 * 520 + 515, dtype=io, device=dev), torch.zeros(135 * 520 + 515, dtype=io, device=dev)
        vx, vw = sx.as_strided((70, 515), (520, 1)), sw.as_strided((136, 515), (520, 1))
        vx.copy_(x)
        vw.copy_(w)
        sx.as_strided((69, 5), (520, 1), 515).fill_(float("nan"))   # between the rows
        sw.as_strided((135, 5), (520, 1), 515).fill_(float("nan"))
        check(vx, vw, b, "silu", r, dy)
        check(vx[:9], vw, b, "silu", r[:9], dy[:9])


@pytest.mark.parametrize("M,N,K", [(70, 65, 4200), (65, 64, 64), (129, 200, 130), (2100, 2050, 72), (3000, 1100, 40), (66, 3000, 1000),
                                   (3700, 3500, 136)])
def test_tiles_and_splits(dev, M, N, K):
    """Every size of tile, ragged in each direction, with one split of k and with several."""
    x, w, b, r, dy = make(dev, (M, K), N, BF16, seed=M)
    check(x, w, b, "gelu", r, dy)


@pytest.mark.parametrize("M,N,K", [(3700, 3500, 400), (1800, 2000, 272), (700, 130, 4112)])
def test_8bit_tiles(dev, M, N, K):
    """Whole numbers (exact sums) through every size of tile."""
    r = torch.Generator().manual_seed(10)
    x, w = (torch.randint(-4, 5, s, generator=r).float() for s in ((M, K), (N, K)))
    ones = torch.ones(max(M, N), device=dev) / 64
    y = ssm_scan.linear_8bit(x.to(torch.float8_e4m3fn).to(dev), ones[:M], w.to(torch.float8_e4m3fn).to(dev), ones[:N])
    assert torch.equal(y.cpu(), (x.to(dev) @ w.to(dev).t() / 4096).bfloat16().cpu())
