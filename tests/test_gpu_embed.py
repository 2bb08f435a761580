"""The token embedding and its gradient against the float64 oracle (oracle/token_ref.py).

Tolerances.  Forward: the product's rounding in float32 and half a step (below the smallest normal number, that number's).  Gradient: a token's rows are added one after
the other within pieces of 32, pieces and groups likewise, so a sum of c terms is off by c roundings of float32 of the
terms' magnitudes at most, and two more for the scale."""

import math

import pytest
import torch

from oracle import token_ref
import ssm_scan
from ssm_scan import linear

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def check(tokens, w, scale, dout):
    leaf = w.detach().requires_grad_()
    out = ssm_scan.embedding(tokens, leaf, scale=scale)
    assert out.dtype == w.dtype and out.shape == tokens.shape + (w.shape[1],)
    want, dw, mag = token_ref.embedding(tokens, w, scale, dout)
    half = torch.finfo(w.dtype).eps / 2
    got = out.detach().double().cpu().reshape(want.shape)
    assert ((got - want).abs() <= half * want.abs().clamp(min=torch.finfo(w.dtype).tiny) + 2.0 ** -23 * want.abs()).all()
    g, = torch.autograd.grad(out, leaf, dout)
    assert g.dtype == w.dtype and g.shape == w.shape
    count = torch.bincount(tokens.cpu().reshape(-1).long().clamp(-1, w.shape[0]) + 1, minlength=w.shape[0] + 2)[1:-1]
    tol = half * dw.abs().clamp(min=torch.finfo(w.dtype).tiny) + (count[:, None] + 3) * 2.0 ** -24 * mag
    off = (g.double().cpu() - dw).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.3g} x"


def make(dev, n, V, D, io, kind, seed=0):
    r = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        tokens = torch.randint(0, V, (n,), generator=r)
    elif kind == "one":
        tokens = torch.full((n,), V // 2)
    elif kind == "frequent":   # ranks by 1 / rank
        tokens = torch.exp(torch.rand(n, generator=r) * math.log(V + 1)).long().sub(1).clamp(0, V - 1)
        tokens = torch.randperm(V, generator=r)[tokens]
    else:                      # ids outside the vocabulary among them
        tokens = torch.randint(-3, V + 4, (n,), generator=r)
        tokens[::7] = torch.tensor([-1, V, 2 ** 40, -(2 ** 60), 2 ** 32])[torch.arange(len(tokens[::7])) % 5]
    return tokens.to(dev), (0.05 * torch.randn(V, D, generator=r)).to(io).to(dev), torch.randn(n, D, generator=r).to(io).to(dev)


# one token and channel; rows that fill no load; vocabularies of one, two and three sorting passes and at their borders;
# runs that end inside, at and past a piece; more tokens than the sort has wavefronts' steps
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("n,V,D,kind", [(1, 1, 1, "one"), (1, 5, 8, "uniform"), (63, 3, 16, "uniform"), (64, 2, 24, "one"), (65, 1, 40, "one"),
                                        (128, 511, 64, "one"), (129, 512, 64, "outside"), (500, 256, 100, "frequent"),
                                        (4096, 256, 32, "frequent"), (8192, 1000, 256, "frequent"), (3000, 70000, 12, "frequent"),
                                        (2500, 300000, 8, "outside"), (20000, 50001, 64, "frequent"), (700, 40, 33, "outside"),
                                        (300, 10, 2056, "uniform"), (9000, 7, 520, "uniform")])
def test_sizes(dev, io, n, V, D, kind):
    tokens, w, dout = make(dev, n, V, D, io, kind, seed=n + V)
    check(tokens, w, 1.0, dout)
    check(tokens, w, -7.3, dout)


@pytest.mark.parametrize("kind", ["one", "frequent", "uniform", "outside"])
def test_long_batches(dev, kind):
    """From 2^15 tokens on, sums of groups of pieces are formed too."""
    tokens, w, dout = make(dev, 150001, 9, 16, F32, kind)
    check(tokens, w, 0.5, dout)


def test_shapes_types_and_strides(dev):
    tokens, w, dout = make(dev, 60, 50, 64, BF16, "outside", seed=3)
    t3 = tokens.reshape(3, 4, 5)
    check(t3, w, 2.0, dout.reshape(3, 4, 5, 64))
    ref = ssm_scan.embedding(tokens, w, 2.0)
    small = tokens.clamp(-1, 50)
    assert torch.equal(ssm_scan.embedding(small.int(), w, 2.0), ssm_scan.embedding(small, w, 2.0))
    assert torch.equal(ssm_scan.embedding(torch.stack([tokens, tokens], 1)[:, 0], w, 2.0), ref)
    wide = torch.cat([w[:, :3], w, w], 1)
    assert torch.equal(ssm_scan.embedding(tokens, wide[:, 3:67], 2.0), ref)      # rows at no whole load
    assert torch.equal(ssm_scan.embedding(tokens, w.t().contiguous().t(), 2.0), ref)
    leaf = w.detach().requires_grad_()
    g, = torch.autograd.grad(ssm_scan.embedding(tokens, leaf, 2.0), leaf, dout)
    g2, = torch.autograd.grad(ssm_scan.embedding(tokens, leaf, 2.0), leaf, torch.cat([dout, dout], 1)[:, 64:])
    g3, = torch.autograd.grad(ssm_scan.embedding(tokens, leaf, 2.0), leaf, torch.cat([dout[:, :1], dout], 1)[:, 1:])
    g4, = torch.autograd.grad(ssm_scan.embedding(tokens, leaf, 2.0), leaf, dout[:1].expand(60, 64))
    assert torch.equal(g, g2) and torch.equal(g, g3)
    assert torch.equal(g4, torch.autograd.grad(ssm_scan.embedding(tokens, leaf, 2.0), leaf, dout[:1].repeat(60, 1))[0])


def test_repeatable_and_captured(dev):
    """The same bits every time, in a captured step too, which takes the tokens of its replay."""
    tokens, w, dout = make(dev, 5000, 300, 64, F32, "frequent", seed=4)
    leaf = w.requires_grad_()

    def step():
        out = ssm_scan.embedding(tokens, leaf, 3.0)
        return out.detach(), torch.autograd.grad(out, leaf, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, g = step()
    for k in range(3):
        tokens.copy_(torch.roll(tokens, 17 * k + 1) if k else tokens)
        graph.replay()
        torch.cuda.synchronize()
        want, gw = step()
        assert torch.equal(out, want) and torch.equal(g, gw), k


def test_refusals_and_no_tokens(dev):
    w = torch.zeros(10, 16, device=dev)
    t = torch.zeros(4, dtype=torch.long, device=dev)
    with pytest.raises(TypeError):
        ssm_scan.embedding(t.float(), w)
    with pytest.raises(TypeError):
        ssm_scan.embedding(t, w.double())
    with pytest.raises(ValueError):
        ssm_scan.embedding(t, w[0])
    with pytest.raises(ValueError):
        ssm_scan.embedding(t, w[:0])
    with pytest.raises(ValueError):
        ssm_scan.embedding(t, w, scale=float("inf"))
    leaf = w.clone().requires_grad_()
    e = ssm_scan.embedding(t[:0].reshape(2, 0), leaf)
    assert e.shape == (2, 0, 16) and not torch.autograd.grad(e.sum(), leaf)[0].any()


@pytest.mark.parametrize("V,n", [(10, 60), (5000, 300)])
def test_derivatives_of_the_gradient(dev, V, n):
    """Of sum of out^3: the terms of a row and channel are alike, so n additions and fewer than 16 other roundings of
    float32 are off by n + 16 halves of its step, relative to the result."""
    tokens, w, _ = make(dev, n, V, 24, F32, "uniform", seed=6)
    tokens, r = tokens.clamp(0, V - 1), torch.randn(V, 24, generator=torch.Generator().manual_seed(7)).to(dev)

    def twice(call, w, r):
        leaf = w.detach().requires_grad_()
        g, = torch.autograd.grad((call(leaf) ** 3).sum(), leaf, create_graph=True)
        return torch.autograd.grad((g * r).sum(), leaf)[0]

    want = twice(lambda leaf: 1.5 * leaf[tokens], w.double(), r.double())
    layer = torch.nn.Embedding(V, 24).to(dev)
    layer.weight = torch.nn.Parameter(w.detach())
    got = twice(lambda leaf: ssm_scan.embedding(tokens, leaf, 1.5), w, r)
    assert ((got - want).abs() <= (n + 16) * 2.0 ** -24 * want.abs()).all()
    if V > 4096:   # a layer of a model
        g, = torch.autograd.grad((linear.embedding(layer, tokens) ** 3).sum(), layer.weight, create_graph=True)
        got, = torch.autograd.grad((g * r).sum(), layer.weight)
        assert ((1.5 ** 3 * got - want).abs() <= (n + 18) * 2.0 ** -24 * want.abs()).all()


def test_forward_mode_of_a_layer(dev):
    layer = torch.nn.Embedding(5000, 16).to(dev)
    tokens, tangent = torch.arange(40, device=dev), torch.randn(5000, 16, device=dev)
    with torch.autograd.forward_ad.dual_level():
        w = torch.autograd.forward_ad.make_dual(layer.weight.detach(), tangent).requires_grad_()
        del layer.weight
        layer.weight = w
        out = torch.autograd.forward_ad.unpack_dual(linear.embedding(layer, tokens))
    assert torch.equal(out.tangent, tangent[:40])
