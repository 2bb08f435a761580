"""The gated delta rule's walks where a wavefront takes two tiles of 16 columns of v (more than 256 tiles over
all heads), and over many chunks, against the float64 oracle with test_gpu_delta's tolerances."""

import pytest
import torch

import ssm_scan
from test_gpu_delta import BF16, F16, F32, check, close, make
from oracle import delta_ref

pytestmark = pytest.mark.gpu


def tiles(B, L, Hk, H, Dk, Dv):
    return B * H * -(-Dv // 16)


# both key widths; an even and an odd count of tiles, a last tile that is not full, unaligned rows; heads that
# are a multiple of 8 and not; shared keys and not; a length that ends inside a chunk
PAIRS = [(8, 130, 8, 8, 64, 80), (8, 70, 4, 8, 128, 72), (11, 65, 3, 9, 40, 34), (5, 150, 13, 13, 100, 64), (9, 200, 1, 3, 80, 170)]


@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("shape", PAIRS)
def test_pairs_of_tiles_match_the_oracle(dev, shape, io):
    assert tiles(*shape) > 256
    a, do, dl = make(dev, *shape, io, seed=21)
    check(a, do, dl, io, True)


@pytest.mark.parametrize("io", [F32, BF16, F16])
def test_pairs_of_tiles_without_norm_state_or_last(dev, io):
    shape = (16, 90, 2, 4, 48, 66)
    assert tiles(*shape) > 256
    a, do, dl = make(dev, *shape, io, seed=22, norm=False, strided=True, beta_type=F32)
    a["h0"] = None
    check(a, do, dl, io, False, scale=0.3, last=False)


def test_pairs_and_single_tiles_agree_bit_for_bit(dev):
    """The columns of v do not mix: a row of a batch alone (single tiles) gives what it gives within the batch."""
    shape = (40, 140, 2, 4, 64, 48)
    assert tiles(*shape) > 256 >= tiles(1, *shape[1:])
    a, do, dl = make(dev, *shape, F32, seed=23)
    a = {n: t.requires_grad_() for n, t in a.items()}

    def once(x, do, dl):
        o, s = ssm_scan.gated_delta_rule(**x, qk_norm=True, return_last_state=True)
        return [o, s] + list(torch.autograd.grad([o, s], list(x.values()), [do, dl]))

    whole = once(a, do, dl)
    for b in (0, 39):
        alone = once({n: t[b:b + 1].detach().requires_grad_() for n, t in a.items()}, do[b:b + 1], dl[b:b + 1])
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(whole, alone))


@pytest.mark.parametrize("io,shape", [(F32, (1, 1500, 1, 2, 64, 32)), (BF16, (1, 1100, 2, 2, 128, 40)), (F16, (2, 961, 1, 3, 30, 50))])
def test_many_chunks(dev, io, shape):
    a, do, dl = make(dev, *shape, io, seed=24)
    check(a, do, dl, io, True)


def test_a_decay_with_nothing_before_it_over_pairs(dev):
    a, do, _ = make(dev, 16, 64, 4, 4, 64, 80, F32, seed=25)
    a["h0"] = None
    g = a["g"].requires_grad_()
    o = ssm_scan.gated_delta_rule(**a, qk_norm=True)
    d = torch.autograd.grad(o, g, do)[0]
    _, _, want = delta_ref.delta(**a, qk_norm=True, dout=do)
    close("dg", d, want["g"], F32, grad=True)
