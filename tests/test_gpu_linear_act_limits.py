"""The linear layer at the ends of its range: rows whose tiles pass 32-bit offsets, arguments of the activation beyond the
operands' type, operands whose rows share their memory, scales whose product leaves float32, GELU's tail, operands of one
channel with any stride."""

import pytest
import torch

import ssm_scan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("MN,K", [(3331, 4300000), (1800, 8500000)])
def test_long_rows(dev, MN, K):
    """Row 255 (or 127) of a tile begins more than 2^31 bytes after its first.  Small whole numbers at both ends of the rows:
    sums are exact."""
    if torch.cuda.mem_get_info()[0] < 5 * MN * K:
        pytest.skip("not enough memory")
    r = torch.Generator().manual_seed(1)
    cols = torch.cat([torch.arange(64), torch.arange(K - 64, K)]).to(dev)
    x, w = (torch.zeros(MN, K, dtype=BF16, device=dev) for _ in range(2))
    small = [torch.randint(-2, 3, (MN, 128), generator=r).to(dev).float() for _ in range(2)]
    for t, s in zip((x, w), small):
        t[:, :64] = s[:, :64].to(BF16)
        t[:, -64:] = s[:, 64:].to(BF16)
    y = ssm_scan.linear_act(x, w)
    assert len(cols) == 128 and torch.equal(y, (small[0] @ small[1].t()).to(BF16))
    del x, w, t
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_where_z_leaves_float16(dev, act):
    """z = -10^5, which float16 keeps as -inf: the activation and its slope are 0.  z = 10^5: the slope is 1."""
    x = torch.tensor([[1000.0], [-1000.0], [1.0]], device=dev, dtype=F16).requires_grad_()
    w = torch.tensor([[-100.0], [0.5]], device=dev, dtype=F16).requires_grad_()
    b = torch.zeros(2, device=dev, dtype=F16).requires_grad_()
    y = ssm_scan.linear_act(x, w, b, act)
    assert y[0, 0] == 0 and y[1, 0] == float("inf")
    dy = torch.tensor([[2.0, 1.0], [4.0, 1.0], [0.0, 0.0]], device=dev, dtype=F16)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    # slopes: 0 and 1 (z = 500) of the first row, 1 and 0 (z = -500) of the second
    assert torch.equal(dx.cpu(), torch.tensor([[0.5], [-400.0], [0.0]], dtype=F16))
    assert torch.equal(dw.cpu(), torch.tensor([[-4000.0], [1000.0]], dtype=F16))
    assert torch.equal(db.cpu(), torch.tensor([4.0, 1.0], dtype=F16))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_of_not_a_number(dev, act):
    x = torch.tensor([[float("nan")], [2.0]], device=dev, dtype=BF16).requires_grad_()
    w = torch.ones(3, 1, device=dev, dtype=BF16)
    dx, = torch.autograd.grad(ssm_scan.linear_act(x, w, activation=act), x, torch.ones(2, 3, device=dev, dtype=BF16))
    assert torch.isnan(dx[0]).all() and torch.isfinite(dx[1]).all()


@pytest.mark.parametrize("M", [70, 200, 300])
def test_infinities_in_rows_that_share_their_memory(dev, M):
    """Broadcast rows of x (in dweight) and of weight (in dx): the sum ends with the last row."""
    row = torch.ones(1, 256, device=dev, dtype=BF16)
    row[0, 5] = float("inf")
    other = torch.ones(72, 256, device=dev, dtype=BF16)
    w = other.clone().requires_grad_()
    y = ssm_scan.linear_act(row.expand(M, 256), w)
    g, = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.full((72, 256), float(M), device=dev)
    want[:, 5] = float("inf")
    assert torch.equal(g.float(), want.to(BF16).float())
    x = other.clone().requires_grad_()
    y = ssm_scan.linear_act(x, row.expand(M, 256))
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(g.float(), want.to(BF16).float())


def test_overlapping_rows(dev):
    """Rows that begin 8 elements apart: a window over one signal."""
    signal = torch.randn(8 * 69 + 256, device=dev).to(BF16)
    x = signal.as_strided((70, 256), (8, 1))
    w, dy = torch.randn(40, 256, device=dev).to(BF16), torch.randn(70, 40, device=dev).to(BF16)
    got = []
    for t in (x, x.contiguous()):
        leaf = w.clone().requires_grad_()
        y = ssm_scan.linear_act(t, leaf)
        got.append([y.detach(), *torch.autograd.grad(y, leaf, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("M", [3, 70])
def test_8bit_scales_whose_product_leaves_float32(dev, M):
    """The product of the scales alone would be of a few bits, 0 or infinite; the result is none of them.  The largest values: sums
    are 49 2^21 or 0, exactly, two roundings of float32 and half a step of bfloat16 remain."""
    K = 512
    q = torch.full((M, K), 448.0, device=dev)
    wq = torch.full((16, K), 448.0, device=dev)
    wq[1::4, ::2] = -448.0     # sums of zero
    for xs, ws in ((1.3e-25, 1.7e-20), (1.1e-30, 1.9e-12), (3e-38, 1.5e-7), (1.3e25, 1.7e-20), (1.3e20, 1.1e16), (5e30, 7e20)):
        y = ssm_scan.linear_8bit(q.to(torch.float8_e4m3fn), torch.full((M,), xs, device=dev), wq.to(torch.float8_e4m3fn), torch.full((16,), ws, device=dev))
        z = 448.0 * wq.double().sum(1).cpu() * torch.tensor(xs).double() * torch.tensor(ws).double()
        z = z.expand(M, 16)
        got = y.double().cpu()
        big = z.abs() > torch.finfo(BF16).max
        assert torch.isinf(got[big]).all() and (got[z == 0] == 0).all(), (xs, ws)
        tol = 2.0 ** -8 * z.abs().clamp(min=torch.finfo(BF16).tiny) + 3 * 2.0 ** -24 * z.abs()
        assert ((got - z).abs()[~big] <= tol[~big]).all(), (xs, ws)


@pytest.mark.parametrize("io", [BF16, F16])
def test_gelu_tail(dev, io):
    """z Phi(z) and its slope for z from -12 to 12, z exact.  A relative error e of erfc's argument is one of z^2 e of Phi (and of
    the density): e is at most three roundings, and as many again follow, so (z^2 + 4) 2^-22 of each term; then half a step of
    the result, and for the slope, which is rounded as dz and as dx (weights of one), twice."""
    z = torch.cat([torch.linspace(-12, 12, 2001), torch.tensor([-5.0, -5.5, -0.0, 0.0])]).to(io)[:, None]
    x = z.to(dev).requires_grad_()
    y = ssm_scan.linear_act(x, torch.ones(1, 1, device=dev, dtype=io), activation="gelu")
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    v = z.double()
    half, tiny = torch.finfo(io).eps / 2, torch.finfo(io).tiny
    phi, density = 0.5 * torch.erfc(-v * 0.5 ** 0.5), torch.exp(-0.5 * v * v) / (2 * torch.pi) ** 0.5
    want, slope = v * phi, phi + v * density
    grow = (v * v + 4) * 2.0 ** -22
    assert ((y.detach().double().cpu() - want).abs() <= half * want.abs().clamp(min=tiny) + grow * want.abs()).all()
    tol = 2 * half * slope.abs().clamp(min=tiny) * (1 + half) + grow * (phi + (v * density).abs())
    assert ((g.double().cpu() - slope).abs() <= tol).all()


def test_one_channel_with_any_stride(dev):
    """(n, 1) tensors whose last stride is n: transposed rows, and what autograd makes of them."""
    x, w, r, dy = (torch.randn(1, n, device=dev).to(BF16).t() for n in (5, 7, 5, 5))
    assert x.stride() == (1, 5)
    assert torch.equal(ssm_scan.linear_act(x, w), ssm_scan.linear_act(x.clone(memory_format=torch.contiguous_format).reshape(5).reshape(5, 1), w.reshape(7).reshape(7, 1)))
    X, W = torch.randn(5, 16, device=dev).to(BF16).requires_grad_(), torch.randn(1, 16, device=dev).to(BF16).requires_grad_()
    y = ssm_scan.linear_act(X, W, residual=r)
    assert torch.equal(y, ssm_scan.linear_act(X, W, residual=r.reshape(5).reshape(5, 1)))
    a = torch.autograd.grad(ssm_scan.linear_act(X, W, residual=r), [X, W], dy)
    b = torch.autograd.grad(ssm_scan.linear_act(X, W, residual=r), [X, W], dy.reshape(5).reshape(5, 1))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    (ssm_scan.linear_act(X, W).t().float() @ torch.randn(5, 3, device=dev)).sum().backward()
    assert torch.isfinite(X.grad).all()
    q, s = ssm_scan.quantize_rows(x.float())
    wq, ws = ssm_scan.quantize_rows(w.float())
    flat = lambda t: t.view(torch.uint8).reshape(-1).clone().reshape(-1, 1).view(torch.float8_e4m3fn)
    turned = lambda t: t.view(torch.uint8).reshape(1, -1).t().view(torch.float8_e4m3fn)
    assert torch.equal(ssm_scan.linear_8bit(turned(q), s, turned(wq), ws), ssm_scan.linear_8bit(flat(q), s, flat(wq), ws))
