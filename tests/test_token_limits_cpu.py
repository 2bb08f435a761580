"""CPU tier of the operators around the mixers at the ends of their ranges: the linear layer's plan where rows are long, the
checks that come before anything reaches the device."""

import ctypes
import math

import pytest
import torch
import torch.nn as nn

from oracle import token_ref
from ssm_scan import _abi, linear
from test_token_cpu import embed, linear as linear_args, rnorm, sample


def product(m, n, k, in8=0, stride=None):
    t = _abi.Tensor(4096, (ctypes.c_int64 * 3)(stride or k, 1, 0))
    return _abi.LinearArgs(m=m, n=n, k=k, dtype=_abi.BF16, x=t, weight=t, in8=in8, x_scale=4096, weight_scale=4096)


@pytest.mark.parametrize("in8", [0, 1])
def test_tiles_of_long_rows_stay_within_32_bits(in8):
    """A tile's loads take offsets below 2^31 from its first row, whether the rows are read in place or copied."""
    lib, seen, e = _abi.lib(), set(), 1 if in8 else 2
    for k in [1 << b for b in range(10, 25)] + [4210000, 4210752, 4300000, 5160000, 8454000, 8500000, 16777208]:
        for m, n in [(40, 1 << 10), (64, 64), (1000, 1000), (1024, 1024), (1800, 1800), (2040, 2040), (3331, 3331), (3584, 3584), (8192, 8192), (3400, 4080)]:
            if max(m, n) * k > 1 << 34:
                continue
            tile = lib.ssm_linear_tile(ctypes.byref(product(m, n, k, in8)))
            assert tile in (0, 64, 128, 256)
            if tile:
                assert (tile - 1) * k * e + 512 < 1 << 31, (m, n, k, tile)
                seen.add(tile)
                for stride in (k + 3, 1 << 22, 1 << 23):   # copied, or read where their own stride allows it
                    assert lib.ssm_linear_tile(ctypes.byref(product(m, n, k, in8, max(stride, k)))) in (0, tile)
            if k % 16 == 0 and k * e >= 1 << 22:   # as long as a copy would be: nothing is copied, sums of splits at most
                assert lib.ssm_linear_workspace_bytes(ctypes.byref(product(m, n, k, in8))) <= m * n * 4 * 512, (m, n, k)
    assert seen == {64, 128, 256}
    assert lib.ssm_linear_tile(ctypes.byref(product(8192, 8192, 2048, in8))) == 256
    assert lib.ssm_linear_tile(ctypes.byref(product(1, 4096, 1024, in8))) == 0
    assert lib.ssm_linear_tile(ctypes.byref(product(0, 8, 8))) == -1
    # a stride past the reach of the tile is copied
    far = product(8192, 8192, 2048, in8, stride=1 << 24)
    assert lib.ssm_linear_workspace_bytes(ctypes.byref(far)) == 2 * 8192 * 2048 * e


def test_embedding_scales_are_finite_in_float32():
    fn = _abi.lib().ssm_embed_check
    for scale in (1e39, -1e300, math.nan):
        assert fn(ctypes.byref(embed(scale=scale))) == _abi.EINVAL
    assert fn(ctypes.byref(embed(scale=-3e38))) == _abi.OK


def test_the_oracles_min_p_above_one_keeps_the_first():
    logits = torch.tensor([[0.0, 1.0, 1.0, 0.5]])
    for u in (0.0, 0.6, 0.99):
        assert token_ref.sample(logits, torch.tensor([u]), min_p=1.5)[0][0] == 1
        assert token_ref.sample(logits, torch.tensor([u]), min_p=1.0)[0][0] == (1 if u < 0.5 else 2)


def test_layers_that_may_be_passed_by():
    layer = nn.Embedding(10, 4)
    assert linear.plain_call(layer, nn.Embedding)
    for register in (layer.register_forward_hook, layer.register_forward_pre_hook, layer.register_full_backward_hook,
                     layer.register_full_backward_pre_hook):
        h = register(lambda *a: None)
        assert not linear.plain_call(layer, nn.Embedding)
        h.remove()
        assert linear.plain_call(layer, nn.Embedding)
    h = nn.modules.module.register_module_forward_hook(lambda *a: None)
    assert not linear.plain_call(layer, nn.Embedding)
    h.remove()

    class Own(nn.Embedding):
        pass

    class Weight(nn.Parameter):   # as a distributed tensor's
        pass

    assert not linear.plain_call(Own(10, 4), nn.Embedding)
    layer.weight = Weight(torch.zeros(10, 4))
    assert not linear.plain_call(layer, nn.Embedding)
    layer = nn.Embedding(10, 4)
    layer.forward = lambda i: i
    assert not linear.plain_call(layer, nn.Embedding)
    seen = []
    torch.func.grad(lambda w: (seen.append(linear.plain_call(nn.Embedding(10, 4), nn.Embedding)), w.sum())[1])(torch.ones(3))
    assert seen == [False]


def test_a_trained_layers_ids_are_checked_as_the_layer_does():
    """The node that stands in for a layer looks its rows up with the layer's own function, which refuses other ids."""
    w = torch.randn(5000, 4, requires_grad=True)
    for bad in (-1, 5000):
        with pytest.raises(IndexError):
            _abi.host().embedding_layer(torch.tensor([3, bad]), w)
    idx = torch.tensor([[3, 4999], [0, 3]])
    out = _abi.host().embedding_layer(idx, w)
    assert torch.equal(out, w[idx]) and out.requires_grad


def test_workspaces_are_aligned():
    """Refused before anything reaches the device."""
    lib, t = _abi.lib(), _abi.Tensor(256, (ctypes.c_int64 * 3)(8, 1, 0))
    big = 1 << 40
    for call, args in ((lib.ssm_rnorm_bwd, rnorm(sum=t, dout=t, dx=t, weight=256, dweight=256)),
                       (lib.ssm_embed_bwd, embed(tokens=256, dout=t, dweight=256)),
                       (lib.ssm_linear_fwd, linear_args(m=100, n=4096, k=4096, out=t)),
                       (lib.ssm_linear_bwd, linear_args(dout=t, activation=1, pre=256, dx=t)),
                       (lib.ssm_sample, sample(logits=t, u=256, token=256, logprob=256, vocab=100000))):
        args.workspace_bytes = big
        for at in (257, 260, 264):
            args.workspace = at
            assert call(ctypes.byref(args), None) == _abi.EINVAL and b"aligned" in lib.ssm_last_error()
        args.workspace, args.workspace_bytes = 256, 16
        assert call(ctypes.byref(args), None) == _abi.ESPACE
