"""The draw of the next token against the float64 oracle (oracle/token_ref.py).

Tokens have to be equal: both sides round far below the distance of u from a border (the weights' integers by 2^-44 of
the largest and less).  Log probabilities are a float64 difference rounded once: 2^-24, and 2^-40 for the sum's."""

import math

import numpy as np
import pytest
import torch

from oracle import token_ref
import ssm_scan

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(dev, B, V, io, seed=0, spread=2.0):
    r = torch.Generator().manual_seed(seed)
    logits = spread * torch.randn(B, V, generator=r)
    logits[torch.rand(B, V, generator=r) < 0.03] = -math.inf
    logits[:, V // 2] = 0.5
    return logits.to(io).to(dev), torch.rand(B, generator=r).to(dev)


def check(logits, u, **kw):
    token, logprob = ssm_scan.sample(logits, u, **kw)
    want, lp = token_ref.sample(logits, u, **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert token.dtype == torch.int64 and logprob.dtype == F32 and token.shape == logprob.shape == u.shape
    assert np.array_equal(token.cpu().numpy(), want), (token.cpu().numpy()[token.cpu().numpy() != want], want[token.cpu().numpy() != want])
    got = logprob.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(lp))
    fine = ~np.isnan(lp)
    assert (np.abs(got - lp)[fine] <= 2.0 ** -24 * np.abs(lp[fine]) + 2.0 ** -40 * len(logits[0])).all()
    return token


SETTINGS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=100), dict(top_p=0.9),
            dict(top_p=0.3, temperature=1.5), dict(min_p=0.1), dict(top_k=50, top_p=0.8, min_p=0.02, temperature=0.8),
            dict(top_p=1e-9), dict(min_p=1.0), dict(min_p=3.0), dict(top_p=0.0), dict(top_p=0.999999), dict(top_k=10 ** 9, top_p=1.0, min_p=0.0)]


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("B,V", [(5, 1), (9, 3), (40, 256), (30, 1000), (6, 5003), (4, 50001)])
def test_settings(dev, io, kw, B, V):
    check(*make(dev, B, V, io, seed=V), **kw)


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("B,V", [(2, 131072), (3, 4096), (3, 4097), (7, 8191), (1, 1100001)])
def test_large_vocabularies(dev, io, B, V):
    logits, u = make(dev, B, V, io, seed=V)
    check(logits, u)
    check(logits, u, top_k=V // 3, top_p=0.97, temperature=1.2)


def test_settings_per_row(dev):
    B = 64
    logits, u = make(dev, B, 3001, BF16, seed=7)
    r = torch.Generator().manual_seed(8)

    def choose(values, dtype=F32):
        return torch.tensor(values, dtype=dtype)[torch.randint(len(values), (B,), generator=r)].to(dev)

    kw = dict(temperature=choose([0.0, 0.6, 1.0, 2.0]), top_k=choose([0, 1, 7, 300, 5000], torch.int64), top_p=choose([1.0, 0.9, 0.4]),
              min_p=choose([0.0, 0.05]))
    check(logits, u, **kw)
    check(logits, u, temperature=0.9, top_k=kw["top_k"].int())
    check(logits, u, top_p=kw["top_p"], min_p=0.01)
    odd = dict(temperature=torch.tensor([-1.0, float("nan"), 0.0, 1.0], device=dev), top_k=torch.tensor([-5, 3, 0, 2], device=dev),
               top_p=torch.tensor([2.0, 0.5, float("nan"), 0.0], device=dev), min_p=torch.tensor([-1.0, 0.1, 0.0, float("nan")], device=dev))
    token, _ = ssm_scan.sample(logits[:4], u[:4], **odd)
    first = logits[:4].float().argmax(-1)
    assert torch.equal(token[:3], first[:3])
    assert token[3] == first[3]   # a top_p of 0 keeps the first


@pytest.mark.parametrize("V", [6, 300, 6000])
def test_ties(dev, V):
    """Equal logits: the lower index comes first in the order, and the draw goes by index."""
    logits = torch.zeros(50, V, device=dev)
    logits[:, ::3] = 1.0
    logits[7, :] = -0.0
    logits[7, 1::2] = 0.0       # zeros of both signs tie
    u = torch.linspace(0, 0.9999, 50, device=dev)
    for kw in (dict(), dict(top_k=2), dict(top_k=V // 3 + 2), dict(top_p=0.5), dict(top_k=V - 1, top_p=0.9), dict(min_p=0.5), dict(top_k=V // 2, top_p=0.35)):
        check(logits, u, **kw)


def test_edges_of_u_and_of_rows(dev):
    logits, _ = make(dev, 8, 700, F32, seed=9)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, 0.5, 0.25, 0.75], device=dev)
    check(logits, u.clamp(0, 1), top_k=20)
    check(logits, u.clamp(0, 1))
    a, _ = ssm_scan.sample(logits, u, top_k=20)
    b, _ = ssm_scan.sample(logits, u.clamp(0, 1), top_k=20)
    assert torch.equal(a, b)                                       # outside [0, 1): as its ends
    check(logits, torch.rand(8, dtype=torch.float64, device=dev))
    logits[1] = -math.inf
    logits[2, 30] = float("nan")
    logits[3, 40:43] = math.inf                                    # they share the mass
    logits[4] = -math.inf
    logits[4, 699] = -1e30                                         # one is left
    logits[5] = torch.finfo(F32).min
    u = torch.full((8,), 0.6, device=dev)
    for kw in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.3), dict(top_k=600, top_p=0.9)):
        token = check(logits, u, **kw)
        assert token[1] == -1 and token[2] == -1 and token[4] == 699 and 40 <= token[3] < 43


def test_all_is_kept_and_all_is_one(dev):
    """A row whose one token has all the mass, and rows colder than the smallest weight."""
    logits = torch.full((3, 5000), -100.0, device=dev)
    logits[:, 4321] = 0.0
    u = torch.tensor([0.0, 0.5, 0.999999], device=dev)
    token, lp = ssm_scan.sample(logits, u)
    assert (token == 4321).all() and (lp.abs() < 1e-12).all()
    check(logits, u, temperature=0.01)
    check(logits, u, temperature=1e4)


def test_strided_rows_and_leading_dims(dev):
    logits, u = make(dev, 24, 999, BF16, seed=10)
    want, lp = ssm_scan.sample(logits, u, top_p=0.9)
    both = torch.cat([logits[:, :5], logits, logits], 1)
    for got in (ssm_scan.sample(both[:, 5:1004], u, top_p=0.9), ssm_scan.sample(logits.t().contiguous().t(), u, top_p=0.9),
                ssm_scan.sample(torch.stack([logits, logits], 1)[:, 1], torch.stack([u, u], 1)[:, 0], top_p=0.9)):
        assert torch.equal(got[0], want) and torch.equal(got[1], lp)
    t, p = ssm_scan.sample(logits.reshape(2, 3, 4, 999), u.reshape(2, 3, 4), top_p=0.9)
    assert torch.equal(t, want.reshape(2, 3, 4)) and torch.equal(p, lp.reshape(2, 3, 4))
    t, _ = ssm_scan.sample(logits[0], u[0], top_p=0.9)
    assert t.shape == () and t == want[0]


def test_frequencies(dev):
    """Evenly spread u draw every kept token as often as its probability says, to one draw."""
    logits = torch.tensor([0.0, 1.0, -1.0, 2.0, -math.inf, 0.5], device=dev)
    n = 20000
    u = (torch.arange(n, device=dev, dtype=torch.float64) + 0.5) / n
    token, _ = ssm_scan.sample(logits.expand(n, 6), u, temperature=0.8, top_k=4)
    kept = torch.where(logits >= 0.0, logits, torch.tensor(-math.inf, device=dev)).double()
    want = torch.softmax(kept / 0.8, 0) * n
    assert ((torch.bincount(token, minlength=6).double() - want).abs() <= 1).all()


def test_captured(dev):
    logits, u = make(dev, 16, 20000, BF16, seed=11)
    T = torch.full((16,), 0.8, device=dev)
    run = lambda: ssm_scan.sample(logits, u, temperature=T, top_p=0.9, top_k=500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, lp = run()
    for k in range(3):
        u.copy_(torch.rand(16, generator=torch.Generator().manual_seed(k)))
        T.fill_(0.5 + 0.4 * k)
        graph.replay()
        torch.cuda.synchronize()
        t, p = run()
        assert torch.equal(token, t) and torch.equal(lp, p), k


def test_refusals_and_no_rows(dev):
    logits, u = make(dev, 4, 50, F32)
    for kw in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=-0.5), dict(min_p=-0.5), dict(top_p=float("nan")),
               dict(temperature=torch.ones(3, device=dev)), dict(top_k=torch.ones(4, 1, dtype=torch.long, device=dev))):
        with pytest.raises(ValueError):
            ssm_scan.sample(logits, u, **kw)
        if not isinstance(next(iter(kw.values())), torch.Tensor):
            with pytest.raises(ValueError):
                ssm_scan.sample(logits[:0], u[:0], **kw)
    with pytest.raises(ValueError):
        ssm_scan.sample(logits, u[:3])
    with pytest.raises(ValueError):
        ssm_scan.sample(logits[:, :0], u)
    with pytest.raises(TypeError):
        ssm_scan.sample(logits.double(), u)
    with pytest.raises(TypeError):
        ssm_scan.sample(logits, u.half())
    with pytest.raises(TypeError):
        ssm_scan.sample(logits, u, top_k=torch.ones(4, device=dev))
    with pytest.raises(RuntimeError, match="not differentiable"):
        ssm_scan.sample(logits.clone().requires_grad_(), u)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.sample(logits, u, top_p=torch.ones(4))
    t, p = ssm_scan.sample(logits[:0], u[:0])
    assert t.shape == p.shape == (0,)


@pytest.mark.parametrize("B,V", [(70, 33000), (5, 70001)])   # workgroups of large and of small chunks
def test_settings_per_row_of_long_rows(dev, B, V):
    logits, u = make(dev, B, V, BF16, seed=12)
    r = torch.Generator().manual_seed(13)

    def choose(values, dtype=F32):
        return torch.tensor(values, dtype=dtype)[torch.randint(len(values), (B,), generator=r)].to(dev)

    check(logits, u, temperature=choose([0.0, 0.1, 0.6, 1.0, 2.0]), top_k=choose([0, 1, 7, 300, 5000, 32000], torch.int64),
          top_p=choose([1.0, 0.9, 0.4, 0.999]), min_p=choose([0.0, 0.05]))
    for kw in (dict(temperature=choose([0.0, 0.7])), dict(top_k=choose([0, 1, 50], torch.int64)), dict(top_p=choose([1.0, 0.8])),
               dict(min_p=choose([0.0, 0.1])), dict(temperature=0.0)):
        check(logits, u, **kw)
    logits[1] = -math.inf
    logits[2, 5] = float("nan")
    logits[3] = 0.0      # a bin of the whole row
    logits[4, 100:20000] = 1.0
    check(logits, u)
    check(logits, u, top_k=10000, top_p=0.8)
    check(logits, u, top_p=0.7)


@pytest.mark.parametrize("V", [2000, 9000, 40000])
def test_crowded_bins(dev, V):
    """More logits in one bin of the histogram than are ranked at once, distinct and tied."""
    g = torch.Generator().manual_seed(14)
    logits = (1e-4 * torch.rand(6, V, generator=g)).to(dev)
    logits[2] = torch.round(logits[2] * 3e4) / 3e4
    logits[3:] -= 50.0
    logits[3:, 17] = 0.0
    u = torch.rand(6, generator=g).to(dev)
    for kw in (dict(top_k=V // 2 + 3), dict(top_p=0.6), dict(top_k=V - 100, top_p=0.5), dict(top_k=1200), dict(top_k=V // 2, temperature=1e3)):
        check(logits, u, **kw)


@pytest.mark.parametrize("V", [30, 1000, 3000, 20000, 33000, 131072])
def test_a_token_that_is_all_that_is_kept(dev, V):   # its probability is 1, whatever the weights' scale
    logits, u = make(dev, 3, V, F32, seed=V)
    for kw in (dict(top_k=1), dict(temperature=0.0), dict(top_k=1, temperature=0.6, top_p=0.5, min_p=0.05)):
        assert (ssm_scan.sample(logits, u, **kw)[1] == 0).all()
