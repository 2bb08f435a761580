"""Grouped norm over more rows than the backward has row slots, so that a slot walks several rows, with
test_gpu_group_norm's tolerances (within a slot dw and db are float32 sums, over the slots float64: a slot of
these shapes has at most 6 rows, 6 roundings of 2^-24 beside the 2^-20 allowed)."""

import pytest
import torch

from test_gpu_group_norm import BF16, F16, F32, check, make

pytestmark = pytest.mark.gpu


def slots(R, C):
    """Of a backward over R rows of C channels (2^21 / C, at least one, at most one a row)."""
    return max(1, min(R, (1 << 21) // C))


# 16-byte loads of one and of several pieces a lane, scalar lanes; rows that are no multiple of the slots
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("mode,center", [("gate", False), ("gate", True), ("silu", True), (None, True), (None, False)])
@pytest.mark.parametrize("R,C,groups", [(1500, 4096, 4), (2100, 2048, 16), (5000, 2040, 120)])
def test_several_rows_a_slot(dev, R, C, groups, mode, center, io):
    assert slots(R, C) < R and R % slots(R, C)
    x, w, b, gate, dy = make(dev, (R, C), io, seed=31)
    check(x, groups, w, b, gate if mode == "gate" else None, "silu" if mode == "silu" else None, center, dy)
