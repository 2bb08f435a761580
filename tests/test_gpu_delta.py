"""Gated delta rule kernels against the float64 token-by-token oracle (oracle/delta_ref.py).

Tolerances.  An output in a 16-bit type is off by half a step of its value (eps / 2: 2^-8 for bf16, 2^-11
for fp16) on top of the arithmetic's error.  The arithmetic is a chain of eight tile products (K S, X, T X,
P U, K^T U, and their counterparts in the gradients), summed in float32 over up to 128 terms (2^-20, with
operands off by 2^-24): eight times 2^-20 of the tensor's largest magnitude, 2^-17.  For 16-bit inputs
Q S and P U have operands off by 2^-16, twice that is 2^-15.  Both are doubled for gradients, whose operands are themselves such results.
With qk_norm, dq = (d - q^ (q^.d)) / |q| is the rest of a cancellation (for Dk = 1 all but 1e-6 of d
cancels): its error goes by d / |q|, whose largest entry the oracle gives."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("q", "k", "v", "g", "beta", "h0")


def close(name, got, want, io, grad=False, size=0.0):
    assert got.shape == want.shape, name
    half = torch.finfo(got.dtype).eps / 2
    chain = (2.0 ** -17 if io == F32 else 2.0 ** -15) * (2 if grad else 1)
    got, want = got.detach().double().cpu(), want.double()
    tol = half * want.abs() + (chain + half * chain) * max(want.abs().max().item(), size)
    bad = (got - want).abs() > tol
    assert torch.isfinite(got).all(), name
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / tol).max().item():.3g} x"


def make(dev, B, L, Hk, H, Dk, Dv, io, seed=0, norm=True, beta_type=None, strided=False):
    r = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=r)

    key = 1.0 if norm else Dk ** -0.5
    if strided:   # the parts of one projection
        m = torch.cat([rn(B, L, 2 * Hk * Dk) * key, rn(B, L, H * Dv)], -1).to(io).to(dev)
        q, k, v = m.split([Hk * Dk, Hk * Dk, H * Dv], -1)
        q, k, v = q.unflatten(-1, (Hk, Dk)), k.unflatten(-1, (Hk, Dk)), v.unflatten(-1, (H, Dv))
    else:
        q, k, v = ((rn(B, L, Hk, Dk) * key).to(io).to(dev), (rn(B, L, Hk, Dk) * key).to(io).to(dev),
                   rn(B, L, H, Dv).to(io).to(dev))
    g = (-torch.rand(B, L, H, generator=r) * torch.rand(H, generator=r)).to(dev)
    beta = torch.sigmoid(rn(B, L, H)).to(beta_type or io).to(dev)
    return dict(q=q, k=k, v=v, g=g, beta=beta, h0=rn(B, H, Dk, Dv).to(dev)), rn(B, L, H, Dv).to(io).to(dev), \
        rn(B, H, Dk, Dv).to(dev)


def check(a, do, dl, io, norm, scale=None, last=True):
    a = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
    o, s = ssm_scan.gated_delta_rule(**a, scale=scale, qk_norm=norm, return_last_state=True)
    assert o.dtype == a["v"].dtype and s.dtype == F32
    want_o, want_s, want = delta_ref.delta(**a, scale=scale, qk_norm=norm, dout=do, dlast=dl if last else None)
    close("o", o, want_o, io)
    close("last", s, want_s, io)
    leaves = [a[n] for n in NAMES if a[n] is not None]
    grads = torch.autograd.grad([o, s] if last else [o], leaves, [do, dl] if last else [do])
    for n, d in zip([n for n in NAMES if a[n] is not None], grads):
        assert d.dtype == a[n].dtype
        close("d" + n, d, want[n], io, grad=True, size=want["size"].get(n, 0.0))


# lengths around a chunk of 64, one token, several chunks; widths that fill no tile; shared keys
SHAPES = [(1, 1, 1, 1, 16, 16), (2, 63, 1, 2, 64, 64), (1, 64, 2, 2, 128, 128), (1, 65, 2, 4, 40, 50), (3, 130, 3, 6, 48, 80),
          (1, 200, 1, 3, 100, 200), (2, 7, 2, 2, 1, 1), (1, 70, 1, 1, 127, 17), (8, 64, 1, 1, 33, 8)]


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_oracle(dev, shape, io):
    a, do, dl = make(dev, *shape, io)
    check(a, do, dl, io, True)


@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_without_norm_state_or_last(dev, io):
    a, do, dl = make(dev, 2, 100, 2, 4, 64, 64, io, seed=1, norm=False)
    a["h0"] = None
    check(a, do, dl, io, False, scale=0.3, last=False)


@pytest.mark.parametrize("io,shape", [(BF16, (2, 100, 2, 4, 64, 64)), (BF16, (2, 90, 1, 2, 36, 20)), (F32, (2, 100, 2, 4, 64, 64)),
                                      (F16, (1, 77, 3, 3, 24, 40))])
def test_strided_views_and_float32_beta(dev, io, shape):
    """The parts of one projection, read in place (aligned rows and not); beta float32."""
    a, do, dl = make(dev, *shape, io, seed=2, strided=True, beta_type=F32)
    check(a, do, dl, io, True)
    t = {n: x if n == "h0" else x.transpose(1, 2).contiguous().transpose(1, 2) for n, x in a.items()}   # (B, H, L, D) storage
    o1, o2 = (ssm_scan.gated_delta_rule(**x, qk_norm=True) for x in (a, t))
    assert torch.equal(o1, o2)
    w = {**a, "q": torch.stack([a["q"], a["q"]], -1)[..., 0]}   # a strided last dimension is copied
    assert torch.equal(o1, ssm_scan.gated_delta_rule(**w, qk_norm=True))


@pytest.mark.parametrize("io", [F32, BF16])
def test_resets_strong_decay_and_zero_beta(dev, io):
    """g = -inf and the type's lowest value forget everything before; beta = 0 leaves the state; a token
    of zero keys and queries gives zeros through the norm."""
    a, do, dl = make(dev, 2, 150, 1, 2, 64, 64, io, seed=3)
    a["g"][0, 40] = -float("inf")
    a["g"][0, 64] = -float("inf")
    a["g"][1, 70] = torch.finfo(F32).min
    a["g"][1, 100:120] = -30.0
    a["beta"][0, 10:100] = 0
    a["beta"][1, 128:] = 0
    a["k"][0, 5] = 0
    a["q"][1, 6] = 0
    check(a, do, dl, io, True)
    a["g"][:, 0] = -float("inf")   # nothing of h0 is left
    one = ssm_scan.gated_delta_rule(**a, qk_norm=True)
    a["h0"] = None
    assert torch.equal(one, ssm_scan.gated_delta_rule(**a, qk_norm=True))


def test_all_beta_zero_keeps_the_state(dev):
    a, _, _ = make(dev, 1, 70, 1, 2, 32, 32, F32, seed=4)
    a["beta"].zero_()
    a["g"].zero_()
    _, last = ssm_scan.gated_delta_rule(**a, return_last_state=True)
    assert torch.equal(last, a["h0"])


def test_correlated_keys(dev):
    """Keys that nearly repeat: the triangular system is far from the identity."""
    a, do, dl = make(dev, 1, 128, 1, 2, 64, 64, F32, seed=5)
    a["k"] = a["k"][:, :1].expand(-1, 128, -1, -1) + 0.05 * a["k"]
    a["g"] *= 0.01
    check(a, do, dl, F32, True)


@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_a_decay_with_nothing_before_it_has_no_gradient(dev, io):
    """Without h0 the first token's decay scales zeros: exactly 0, not the rest of a cancellation."""
    for L in (1, 64):
        a, do, _ = make(dev, 2, L, 1, 2, 64, 48, io, seed=13)
        a["h0"] = None
        g = a["g"].requires_grad_()
        o = ssm_scan.gated_delta_rule(**a, qk_norm=True)
        d = torch.autograd.grad(o, g, do)[0]
        _, _, want = delta_ref.delta(**a, qk_norm=True, dout=do)
        if L == 1:
            assert d.abs().max().item() == 0.0
        close("dg", d, want["g"], io, grad=True)


def test_no_tokens(dev):
    a, _, _ = make(dev, 2, 3, 1, 2, 16, 8, F32)
    a = {n: t if n == "h0" else t[:, :0] for n, t in a.items()}
    o, last = ssm_scan.gated_delta_rule(**a, return_last_state=True)
    assert o.shape == (2, 0, 2, 8) and torch.equal(last, a["h0"])
    a["h0"] = None
    assert ssm_scan.gated_delta_rule(**a, return_last_state=True)[1].abs().sum() == 0


def test_pieces_and_steps_continue_each_other(dev):
    """A prompt in pieces of 100, 1, 64 and 35 tokens, then 5 tokens by the step: one call's outputs."""
    a, _, _ = make(dev, 2, 205, 2, 4, 64, 48, F32, seed=6)
    want_o, want_s = delta_ref.delta(**a, qk_norm=True)
    h, outs, t = a["h0"], [], 0
    for n in (100, 1, 64, 35):
        o, h = ssm_scan.gated_delta_rule(*(a[x][:, t:t + n] for x in NAMES[:5]), h0=h, qk_norm=True, return_last_state=True)
        outs.append(o)
        t += n
    for t in range(200, 205):
        outs.append(ssm_scan.gated_delta_step(h, *(a[x][:, t] for x in NAMES[:5]), qk_norm=True)[:, None])
    close("o", torch.cat(outs, 1), want_o, F32, grad=True)
    close("last", h, want_s, F32, grad=True)


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 64), (5, 2, 6, 128, 128), (3, 1, 1, 1, 1), (2, 2, 4, 100, 50), (2, 1, 3, 65, 66),
                                   (70, 1, 2, 33, 7)])
@pytest.mark.parametrize("norm", [False, True])
def test_step_matches_oracle(dev, shape, io, norm):
    """The state is float32 arithmetic over at most 128 terms: 2^-20 of its largest value."""
    B, Hk, H, Dk, Dv = shape
    a, _, _ = make(dev, B, 1, Hk, H, Dk, Dv, io, seed=7, norm=norm)
    want_o, want_s = delta_ref.delta(**a, qk_norm=norm)
    h = a["h0"].clone()
    o = ssm_scan.gated_delta_step(h, *(a[n][:, 0] for n in NAMES[:5]), qk_norm=norm)
    assert o.dtype == io
    close("o", o, want_o[:, 0], F32)
    close("h", h, want_s, F32)


def test_gradient_along_a_direction_matches_differences(dev):
    """The kernels' gradient against central differences of the float64 oracle's loss: the difference's own
    error (1e-9) is nothing beside the gradients' 2^-16 per element, summed over random signs."""
    a, do, dl = make(dev, 1, 90, 1, 2, 32, 24, F32, seed=8)
    a = {n: t.requires_grad_() for n, t in a.items()}
    o, s = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    grads = dict(zip(NAMES, torch.autograd.grad([o, s], [a[n] for n in NAMES], [do, dl])))
    r = torch.Generator().manual_seed(9)
    for n in NAMES:
        d = torch.randn(a[n].shape, generator=r, dtype=torch.float64)

        def loss(e):
            x = {**a, n: a[n].detach().double().cpu() + e * d}
            o, s = delta_ref.delta(**x, qk_norm=True)
            return ((o * do.double().cpu()).sum() + (s * dl.double().cpu()).sum()).item()

        got, diff = (grads[n].double().cpu() * d).sum().item(), (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(got - diff) < 2.0 ** -15 * grads[n].double().cpu().norm().item() * d.norm().item(), n


def test_partial_gradients(dev):
    """Only some inputs need gradients; only the last state or only the outputs are used."""
    a, do, dl = make(dev, 1, 80, 1, 2, 32, 24, F32, seed=10)
    _, _, want = delta_ref.delta(**a, qk_norm=True, dlast=dl)
    a["v"].requires_grad_()
    _, s = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    s.backward(dl)
    close("dv", a["v"].grad, want["v"], F32, grad=True)


def test_backward_is_bitwise_repeatable(dev):
    a, do, dl = make(dev, 2, 200, 2, 6, 64, 80, BF16, seed=11)
    a = {n: t.requires_grad_() for n, t in a.items()}

    def once():
        o, s = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
        return [o, s] + list(torch.autograd.grad([o, s], [a[n] for n in NAMES], [do, dl]))

    first = once()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, once()))


def test_runs_on_the_callers_stream_and_in_a_graph(dev):
    a, do, dl = make(dev, 2, 150, 1, 2, 64, 64, F32, seed=12)
    want, ws = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    step = [a[n][:, 0].contiguous() for n in NAMES[:5]]
    h = a["h0"].clone()
    want_o = ssm_scan.gated_delta_step(h, *step, qk_norm=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o, last = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, want) and torch.equal(last, ws)
    graph, hg = torch.cuda.CUDAGraph(), a["h0"].clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        og, lg = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
        sg = ssm_scan.gated_delta_step(hg, *step, qk_norm=True)
    for _ in range(3):
        hg.copy_(a["h0"])
        og.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(og, want) and torch.equal(lg, ws) and torch.equal(sg, want_o) and torch.equal(hg, h)
        _ = (want * 2).sum().item()


def test_refusals(dev):
    a, _, _ = make(dev, 2, 10, 2, 4, 16, 16, F32)
    bad = [dict(q=a["q"][:, :9]), dict(k=a["k"][..., :8]), dict(v=a["v"][:, :, :3]), dict(g=a["g"][..., :2]), dict(beta=a["beta"][:1]),
           dict(h0=a["h0"][:, :2]), dict(q=a["q"][0])]
    for kw in bad:
        with pytest.raises(ValueError):
            ssm_scan.gated_delta_rule(**{**a, **kw})
    big = torch.zeros(1, 4, 1, 129, device=dev)
    with pytest.raises(ValueError, match="key_dim"):
        ssm_scan.gated_delta_rule(big, big, a["v"][:1, :4, :1], a["g"][:1, :4, :1], a["beta"][:1, :4, :1])
    with pytest.raises(TypeError):
        ssm_scan.gated_delta_rule(**{**a, "v": a["v"].double()})
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_rule(**{**a, "g": a["g"].cpu()})
    one = [a[n][:, 0] for n in NAMES[:5]]
    for h in (a["h0"].bfloat16(), a["h0"].transpose(2, 3), a["h0"][:1]):
        with pytest.raises(ValueError):
            ssm_scan.gated_delta_step(h, *one)
