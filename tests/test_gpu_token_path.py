"""The operators around the mixers run together, as a model uses them: ids, embedding, the residual stream through
norms and mixers, the 8-bit head, the next token.  Checked against the same steps of plain torch operations, and
captured and replayed; and where the package's own models call them."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import token_ref
import ssm_scan
from ssm_scan import block, linear
from ssm_scan.delta_mixer import GatedDeltaMixer

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def stack(dev, layers=2, d=64, vocab=300, dtype=BF16):
    torch.manual_seed(0)
    embed = (0.3 * torch.randn(vocab, d)).to(dtype).to(dev)
    norms = [block.RMSNorm(d).to(dev) for _ in range(layers + 1)]
    mixers = [GatedDeltaMixer(d, heads=2, key_dim=32).to(dev) for _ in range(layers)]
    for m in mixers:   # decays and weights of the norms stay float32
        m.in_proj.to(dtype)
        m.conv.to(dtype)
        m.out_proj.to(dtype)
    return embed, norms, mixers


def run(embed, norms, mixers, tokens, states=None):
    """The stream after the last layer, and its norm."""
    s = ssm_scan.embedding(tokens, embed, scale=math.sqrt(embed.shape[1]))
    y = ssm_scan.rms_norm(s.float(), norms[0].weight).to(s.dtype)
    for i, m in enumerate(mixers):
        out = m(y, None if states is None else states[i])
        y, s = norms[i + 1](out, residual=s)
    return y, s


def plain(embed, norms, mixers, tokens):
    def norm(t, w):
        return t.float() * torch.rsqrt(t.float().pow(2).mean(-1, keepdim=True) + 1e-5) * w

    s = (embed[tokens].float() * math.sqrt(embed.shape[1])).to(embed.dtype)
    y = norm(s, norms[0].weight).to(s.dtype)
    for i, m in enumerate(mixers):
        out = m(y)
        s = (out.float() + s.float()).to(s.dtype)
        y = norm(s, norms[i + 1].weight).to(s.dtype)
    return y, s


def test_training_pass(dev):
    """Values and gradients beside the plain composition's: what differs is the rounding of sums in another order, which
    the 16-bit steps behind it carry on, a few of their half steps (2^-9) of the largest magnitudes in all."""
    embed, norms, mixers = stack(dev)
    tokens = torch.randint(0, 300, (3, 50), device=dev)
    leaves = [embed.requires_grad_(), norms[1].weight, norms[2].weight, mixers[0].in_proj.weight, mixers[1].out_proj.weight, mixers[0].A_log]
    got, want = run(embed, norms, mixers, tokens), plain(embed, norms, mixers, tokens)
    dout = [torch.randn(3, 50, 64, device=dev).to(BF16) for _ in range(2)]
    gg, gw = (torch.autograd.grad(list(o), leaves, dout) for o in (got, want))
    for a, b in list(zip(got, want)) + list(zip(gg, gw)):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.isfinite(a).all()
        assert (a.float() - b.float()).abs().max() <= 16 * 2.0 ** -9 * b.float().abs().max()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_mixer_with_residual(dev, dtype):
    _, _, mixers = stack(dev, dtype=dtype)
    u, r = (torch.randn(2, 9, 64, device=dev).to(dtype).requires_grad_() for _ in range(2))
    got, want = mixers[0](u, residual=r), r + mixers[0](u)
    half = torch.finfo(dtype).eps / 2
    # one rounding of the sum against one of each product and one of the sum
    assert (got - want).abs().max() <= 3 * half * max(want.abs().max(), r.abs().max()) + 1e-5
    g = torch.autograd.grad(got, [u, r], torch.ones_like(got))
    w = torch.autograd.grad(want, [u, r], torch.ones_like(want))
    assert torch.equal(g[1], w[1]) and (g[0].float() - w[0].float()).abs().max() <= 8 * half * w[0].float().abs().max()
    state = mixers[0].init_state(2, dev, dtype)
    with torch.no_grad():
        y = torch.cat([mixers[0](u[:, i:i + 1], state, residual=r[:, i:i + 1]) for i in range(9)], 1)
    assert (y - want).abs().max() <= 16 * half * want.abs().max() + 1e-5


def test_decoding_with_an_8bit_head_captured(dev):
    """Tokens drawn one after the other by a captured step are those of the eager one."""
    B, vocab = 5, 300
    embed, norms, mixers = stack(dev)
    head, head_scale = ssm_scan.quantize_rows(embed)
    u, tok = torch.rand(B, device=dev), torch.randint(0, vocab, (B,), device=dev)
    T = torch.full((B,), 0.9, device=dev)

    def step(states):
        with torch.no_grad():
            s = ssm_scan.embedding(tok[:, None], embed, scale=8.0)
            y = ssm_scan.rms_norm(s.float(), norms[0].weight).to(s.dtype)
            for i, m in enumerate(mixers):
                s = m(y, states[i], residual=s)
                if i + 1 < len(mixers):
                    y = ssm_scan.rms_norm(s.float(), norms[i + 1].weight).to(s.dtype)
            q, scale = ssm_scan.rms_norm_8bit(s[:, 0], norms[-1].weight)
            logits = ssm_scan.linear_8bit(q, scale, head, head_scale)
            nxt, lp = ssm_scan.sample(logits, u, temperature=T, top_p=0.95)
            tok.copy_(nxt)
            return logits, lp

    def fresh():
        return [m.init_state(B, dev, BF16) for m in mixers]

    def reset(states):
        for st in states:
            st.conv.zero_()
            st.delta.zero_()
        tok.copy_(torch.arange(B, device=dev))

    draws = torch.rand(6, B, generator=torch.Generator().manual_seed(3)).to(dev)
    states = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(states)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, lp = step(states)
    reset(states)
    replayed = []
    for d in draws:
        u.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        replayed.append((tok.clone(), logits.clone(), lp.clone()))
    reset(states)
    for d, (t, lo, p) in zip(draws, replayed):
        u.copy_(d)
        a, b = step(states)
        assert torch.equal(tok, t) and torch.equal(a, lo) and torch.equal(b, p)
    # the last step's draw is the one of its logits
    want, _ = token_ref.sample(replayed[-1][1], draws[-1], temperature=T.cpu(), top_p=0.95)
    assert replayed[-1][0].tolist() == want.tolist()


def test_lm_generates_with_top_p(dev):
    lm = block.MambaLM(n_layers=2, d_model=64).to(dev).eval()
    prompt = torch.randint(0, 256, (3, 12), device=dev)
    a = lm.generate(prompt, 8, top_p=0.9, generator=torch.Generator(dev).manual_seed(1))
    b = lm.generate(prompt, 8, top_p=0.9, generator=torch.Generator(dev).manual_seed(1))
    c = lm.generate(prompt, 8, temperature=torch.tensor([0.0, 0.5, 1.0], device=dev), min_p=0.05, top_k=20)
    assert a.shape == c.shape == (3, 20) and torch.equal(a, b) and torch.equal(a[:, :12], prompt) and int(a.max()) < 256
    greedy = lm.generate(prompt, 8, temperature=0.0, top_p=1.0)
    x = prompt
    with torch.no_grad():
        for _ in range(8):   # the whole sequence anew each time: another order of sums, so ties of logits aside
            x = torch.cat([x, lm(x)[:, -1].argmax(-1, keepdim=True)], 1)
    assert (greedy == x).float().mean() > 0.9
    torch.manual_seed(5)
    old = lm.generate(prompt, 8, top_k=10)
    torch.manual_seed(5)
    assert torch.equal(old, lm.generate(prompt, 8, top_k=10))


def test_large_vocabulary_embedding_of_the_lm(dev):
    layer = torch.nn.Embedding(5000, 32).to(dev)
    idx = torch.randint(0, 5000, (4, 100), device=dev)
    dout = torch.randn(4, 100, 32, device=dev)
    out = linear.embedding(layer, idx)
    assert torch.equal(out, layer.weight[idx])
    g, = torch.autograd.grad(out, layer.weight, dout)
    _, want, mag = token_ref.embedding(idx, layer.weight, 1.0, dout)
    assert ((g.double().cpu() - want).abs() <= 2.0 ** -20 * mag).all()
    with torch.no_grad():
        assert torch.equal(linear.embedding(layer, idx), out)


def test_streams_and_threads(dev):
    """Two calls at once on streams of their own, and a call on another stream than its operands'."""
    x, r, w = torch.randn(500, 512, device=dev).to(BF16), torch.randn(500, 512, device=dev).to(BF16), torch.ones(512, device=dev)
    A, W = torch.randn(300, 512, device=dev).to(BF16), torch.randn(256, 512, device=dev).to(BF16)
    logits, u = torch.randn(16, 50000, device=dev), torch.rand(16, device=dev)
    tok, E = torch.randint(0, 700, (2000,), device=dev), torch.randn(700, 512, device=dev).to(BF16).requires_grad_()
    dout = torch.randn(2000, 512, device=dev).to(BF16)

    def calls():
        with torch.no_grad():
            res = [*ssm_scan.add_rms_norm(x, r, w), ssm_scan.linear_act(A, W, activation="gelu"), *ssm_scan.sample(logits, u, top_p=0.9)]
        res.append(torch.autograd.grad(ssm_scan.embedding(tok, E), E, dout)[0])
        return res

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    for res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    d1 = torch.device("cuda", 1)
    x, w = torch.randn(4, 64, device=d1), torch.ones(64, device=d1)
    y, s = ssm_scan.add_rms_norm(x, x, w)
    assert y.device == d1 and torch.cuda.current_device() == 0
    with pytest.raises(ValueError):
        ssm_scan.add_rms_norm(x, x, w.to("cuda:0"))
