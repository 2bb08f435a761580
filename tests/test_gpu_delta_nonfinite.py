"""Infinities and NaN in the gated delta rule go where the recurrence takes them and nowhere else: what the oracle
has finite is finite and right (test_gpu_delta's tolerances), what it has infinite or NaN is not finite."""

import pytest
import torch

from oracle import delta_ref
import ssm_scan
from test_gpu_delta import BF16, F16, F32, make

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def same(name, got, want, io, grad=False):
    got, want = got.detach().double().cpu(), want.double()
    finite = torch.isfinite(want)
    wrong = torch.isfinite(got) != finite
    assert not wrong.any(), f"{name}: {int(wrong.sum())} of {got.numel()}, first at {wrong.nonzero()[0].tolist()}"
    got, want = got[finite], want[finite]
    if not want.numel():
        return
    half = torch.finfo(io).eps / 2
    chain = (2.0 ** -17 if io == F32 else 2.0 ** -15) * (2 if grad else 1)
    tol = half * want.abs() + (chain + half * chain) * want.abs().max()
    assert ((got - want).abs() <= tol).all(), f"{name}: worst {((got - want).abs() / tol).max().item():.3g} x"


def put(a, name, t, bad):
    """`bad` at one element of token t of the first batch row and head."""
    at = (0, t, 0, 3) if a[name].dim() == 4 else (0, t, 0)
    a[name] = a[name].clone()
    a[name][at] = bad
    return a


# tokens at both ends of a chunk, inside its blocks of 16 and 32, in the second chunk and at the end
@pytest.mark.parametrize("t", [0, 5, 40, 63, 64, 107, 149])
@pytest.mark.parametrize("name,bad", [("q", INF), ("q", NAN), ("k", INF), ("k", NAN), ("v", INF), ("v", -INF), ("v", NAN),
                                      ("beta", INF), ("beta", NAN), ("g", INF), ("g", NAN)])
@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_outputs(dev, io, name, bad, t):
    for shape, norm in (((2, 150, 1, 2, 40, 48), True), ((2, 150, 2, 2, 128, 20), False)):
        a, _, _ = make(dev, *shape, io, seed=71, norm=norm)
        put(a, name, t, bad)
        o, last = ssm_scan.gated_delta_rule(**a, qk_norm=norm, return_last_state=True)
        want_o, want_last = delta_ref.delta(**a, qk_norm=norm)
        assert torch.isfinite(want_o[0, :t]).all()   # nothing before the token hangs on it
        same("o", o, want_o, io)
        same("last", last, want_last, F32 if io == F32 else BF16)


@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_outputs_over_pairs_of_tiles(dev, io):
    """More than 256 column tiles; a padded end of NaN in every operand, another length for every batch row."""
    B, L, H = 14, 130, 4
    a, _, _ = make(dev, B, L, 2, H, 64, 72, io, seed=72)
    lengths = [1, 2, 15, 16, 17, 31, 33, 47, 63, 64, 65, 100, 129, 130]
    for b, n in enumerate(lengths):
        for x in ("q", "k", "v", "g", "beta"):
            a[x][b, n:] = NAN
    o = ssm_scan.gated_delta_rule(**a, qk_norm=True)
    want, _ = delta_ref.delta(**a, qk_norm=True)
    assert all(torch.isfinite(want[b, :n]).all() for b, n in enumerate(lengths))
    same("o", o, want, io)


def test_a_state_that_is_not_finite_stays_in_its_columns(dev):
    a, _, _ = make(dev, 2, 150, 1, 2, 64, 40, F32, seed=73)
    a["h0"][0, 0, 7, 11] = INF
    a["h0"][1, 1, 0, 39] = NAN
    o, last = ssm_scan.gated_delta_rule(**a, qk_norm=True, return_last_state=True)
    want_o, want_last = delta_ref.delta(**a, qk_norm=True)
    same("o", o, want_o, F32)
    same("last", last, want_last, F32)


# one element of token t of the first batch row and head in an operand or the outputs' gradient; the first and last
# tokens of a chunk and of its blocks of 16 and 32, a second chunk, the end
@pytest.mark.parametrize("t", [0, 5, 31, 40, 63, 64, 107, 149])
@pytest.mark.parametrize("name,bad", [("q", INF), ("q", NAN), ("k", INF), ("k", NAN), ("v", INF), ("v", NAN), ("beta", NAN), ("do", INF), ("do", NAN)])
@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_gradients(dev, io, name, bad, t):
    for shape, norm in (((2, 150, 1, 2, 128, 20), False), ((2, 150, 2, 2, 40, 48), name in ("v", "do"))):
        a, do, dl = make(dev, *shape, io, seed=74, norm=norm)
        if name == "do":
            do[0, t, 0, 3] = bad
        else:
            put(a, name, t, bad)
        a = {n: x.requires_grad_() for n, x in a.items()}
        o, last = ssm_scan.gated_delta_rule(**a, qk_norm=norm, return_last_state=True)
        grads = torch.autograd.grad([o, last], list(a.values()), [do, dl])
        _, _, want = delta_ref.delta(**a, qk_norm=norm, dout=do, dlast=dl)
        for n, d in zip(a, grads):
            same("d" + n, d, want[n], io if d.dtype == io else BF16 if io == BF16 else F16, grad=True)


def test_gradients_over_pairs_of_tiles(dev):
    """Rows of several lengths whose ends hold anything in v and a gradient of zeros: what is before them is right."""
    B, L, H = 14, 130, 4
    a, do, dl = make(dev, B, L, 2, H, 64, 72, F32, seed=75)
    for b, n in enumerate([1, 2, 15, 16, 17, 31, 33, 47, 63, 64, 65, 100, 129, 130]):
        a["v"][b, n:] = NAN
        do[b, n:] = 0
    a = {n: x.requires_grad_() for n, x in a.items()}
    o = ssm_scan.gated_delta_rule(**a, qk_norm=True)
    grads = torch.autograd.grad(o, list(a.values()), do)
    _, _, want = delta_ref.delta(**a, qk_norm=True, dout=do)
    for n, d in zip(a, grads):
        same("d" + n, d, want[n], F32, grad=True)
