"""linear.embedding(layer, ids): where it stands in for nn.Embedding, the layer's own call keeps what it does: hooks, an
overridden forward, transforms, autocast, the check of the ids."""

import pytest
import torch
import torch.nn as nn

from ssm_scan import _abi, linear

pytestmark = pytest.mark.gpu


def layer(dev, V=5000, D=16, cls=nn.Embedding, dtype=torch.float32):
    torch.manual_seed(0)
    return cls(V, D).to(dev).to(dtype)


def test_hooks_run(dev):
    idx = torch.randint(0, 5000, (40, 30), device=dev)
    for dtype in (torch.float32, torch.bfloat16):
        m = layer(dev, dtype=dtype)
        want = linear.embedding(m, idx)
        seen = []
        h = m.register_forward_hook(lambda mod, args, out: out * 2)
        assert torch.equal(linear.embedding(m, idx), want * 2)
        h.remove()
        h = m.register_forward_pre_hook(lambda mod, args: seen.append(1))
        assert torch.equal(linear.embedding(m, idx), want) and seen == [1]
        h.remove()
        h = m.register_full_backward_hook(lambda mod, gi, go: seen.append(2))
        linear.embedding(m, idx).sum().backward()
        assert seen == [1, 2]
        h.remove()
        assert torch.equal(linear.embedding(m, idx), want)
    h = nn.modules.module.register_module_forward_hook(lambda mod, args, out: out * 3 if mod is m else None)
    try:
        assert torch.equal(linear.embedding(m, idx), want * 3)
    finally:
        h.remove()


class Scaled(nn.Embedding):
    def forward(self, idx):
        return super().forward(idx) * 8.0


def test_a_forward_of_its_own_runs(dev):
    idx = torch.randint(0, 5000, (1200,), device=dev)
    m = layer(dev, cls=Scaled)
    assert torch.equal(linear.embedding(m, idx), m.weight[idx] * 8.0)
    m = layer(dev)
    m.forward = lambda i: nn.Embedding.forward(m, i) + 1.0
    assert torch.equal(linear.embedding(m, idx), m.weight[idx] + 1.0)


class Wrap(nn.Module):
    def __init__(self, m):
        super().__init__()
        self.m = m

    def forward(self, idx):
        return linear.embedding(self.m, idx)


def test_transforms(dev):
    m, idx = Wrap(layer(dev)), torch.tensor([4, 4, 4999], device=dev).repeat(400)
    call = lambda w: torch.func.functional_call(m, {"m.weight": w}, (idx,))
    w = m.m.weight.detach()
    g = torch.func.grad(lambda w: call(w).sum())(w)
    assert g[4].eq(800).all() and g[4999].eq(400).all() and g.sum() == 1200 * 16
    two = torch.stack([w, 2 * w])
    assert torch.equal(torch.func.vmap(call)(two), two[:, idx])


def test_autocast_leaves_small_tables_to_the_layer(dev):
    m, idx = layer(dev, V=100), torch.randint(0, 100, (1200,), device=dev)
    with torch.autocast("cuda", torch.bfloat16):
        out = linear.embedding(m, idx)
    assert out.grad_fn.name() == "EmbeddingBackward0"
    big, idx = layer(dev), torch.randint(0, 5000, (1200,), device=dev)
    with torch.autocast("cuda", torch.bfloat16):
        out = linear.embedding(big, idx)
    assert out.dtype == torch.float32 and out.grad_fn.name() != "EmbeddingBackward0"


@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.int64])
def test_gradient_is_the_sorted_one(dev, idx_dtype):
    m, idx = layer(dev), torch.randint(0, 5000, (4, 700), device=dev).to(idx_dtype)
    dout = torch.randn(4, 700, 16, device=dev)
    import ssm_scan
    w = m.weight.detach().requires_grad_()
    want, = torch.autograd.grad(ssm_scan.embedding(idx, w), w, dout)
    got, = torch.autograd.grad(linear.embedding(m, idx), m.weight, dout)
    assert torch.equal(got, want)
    g, = torch.autograd.grad(linear.embedding(m, idx), m.weight, dout.permute(1, 0, 2).contiguous().permute(1, 0, 2))
    assert torch.equal(g, want)


@pytest.mark.parametrize("dtype,V", [(torch.float32, 5000), (torch.bfloat16, 60)])
def test_lookup_is_the_layers_own(dev, monkeypatch, dtype, V):
    """It checks the ids as the layer in evaluation does; its result can be changed in place."""
    m, idx = layer(dev, V=V, dtype=dtype), torch.randint(0, V, (40, 70), device=dev)
    host, called = _abi.host(), []

    class Spy:
        def __getattr__(self, name):
            called.append(name)
            return getattr(host, name)

    monkeypatch.setattr(_abi, "host", Spy)
    out = linear.embedding(m, idx)
    assert called == ["embedding_layer"] and torch.equal(out, m(idx))
    out += 1
    out.mul_(2)
    g, = torch.autograd.grad(out, m.weight, torch.ones_like(out))
    assert torch.equal(g[:, 0].float(), 2.0 * torch.bincount(idx.reshape(-1), minlength=V))


@pytest.mark.parametrize("n", [1, 1023, 1024])
def test_short_batches_stay_the_layers(dev, n):
    """Below 1024 tokens nn.Embedding's own gradient is faster."""
    m, idx = layer(dev), torch.randint(0, 5000, (n,), device=dev)
    out = linear.embedding(m, idx)
    assert (out.grad_fn.name() == "EmbeddingBackward0") == (n < 1024)
    g, = torch.autograd.grad(out.sum(), m.weight)
    assert torch.equal(g[:, 0], torch.bincount(idx, minlength=5000).float())


def test_derivatives_of_the_layers_gradient(dev):
    """Of sum of out^3 over 1500 tokens: a token's terms are alike, so c of them are off by c + 16 halves of float32's step at most,
    relative to the result; c is below 16 here."""
    m, idx = layer(dev), torch.randint(0, 5000, (1500,), device=dev, generator=torch.Generator(dev).manual_seed(1))
    r = torch.randn(5000, 16, device=dev)
    count = torch.bincount(idx, minlength=5000)
    assert count.max() < 16
    out = linear.embedding(m, idx)
    assert out.grad_fn.name() != "EmbeddingBackward0"
    g, = torch.autograd.grad((out ** 3).sum(), m.weight, create_graph=True)
    got, = torch.autograd.grad((g * r).sum(), m.weight)
    want = 6 * count[:, None].double() * m.weight.detach().double() * r.double()
    assert ((got - want).abs() <= 32 * 2.0 ** -24 * want.abs()).all()
