"""CPU tier: sizes that the gated delta rule refuses because their counts pass what a launch or 64 bits hold."""

import ctypes

import pytest
import torch

import ssm_scan
from ssm_scan import _abi
from test_delta_cpu import delta_args


@pytest.mark.parametrize("kw", [dict(batch=1 << 31, heads=1 << 24, value_dim=1 << 24),   # 2^75 tiles: 0 in 64 bits
                                dict(batch=1 << 40, heads=1 << 24, value_dim=16), dict(batch=1 << 31, heads=4)])
def test_tiles_that_wrap_64_bits(kw):
    lib = _abi.lib()
    for a, check in ((delta_args(**kw), lib.ssm_delta_check), (delta_args(step=True, **kw), lib.ssm_delta_step_check)):
        assert check(ctypes.byref(a)) == _abi.EINVAL and b"too large" in lib.ssm_last_error()


def test_chunks_of_all_heads():
    """What is taken chunk by chunk has up to 512 threads a chunk and head: 2^23 of them are a grid row of 2^32."""
    lib = _abi.lib()
    for L, rc in ((64 * (1 << 19), _abi.EINVAL), (64 * ((1 << 19) - 1), 0)):
        assert lib.ssm_delta_check(ctypes.byref(delta_args(batch=1, heads=16, key_heads=16, seqlen=L))) == rc


def test_keys_of_no_width_are_refused_as_any_other_shape():
    """The default scale, Dk^-0.5, is not formed of a width that the checks refuse."""
    t = torch.zeros
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_rule(t(1, 2, 1, 0), t(1, 2, 1, 0), t(1, 2, 1, 4), t(1, 2, 1), t(1, 2, 1))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_step(t(1, 1, 0, 4), t(1, 1, 0), t(1, 1, 0), t(1, 1, 4), t(1, 1), t(1, 1))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ssm_scan.gated_delta_rule(t(()), t(()), t(()), t(()), t(()))
