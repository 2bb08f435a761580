"""8-bit rows: infinities and NaN as their documentation says, and how far the product adds in steps."""

import pytest
import torch

import ssm_scan

pytestmark = pytest.mark.gpu

F8, INF, NAN = torch.float8_e4m3fn, float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_not_finite_rows(dev, dtype):
    x = torch.ones(4, 40, device=dev, dtype=dtype)
    x[1, 7], x[2, 9], x[3, 1], x[3, 2] = NAN, -INF, INF, NAN
    q, scale = ssm_scan.quantize_rows(x)
    f = q.float()
    at = torch.zeros(4, 40, dtype=torch.bool, device=dev)
    at[1, 7] = at[2, 9] = at[3, 1] = at[3, 2] = True
    assert torch.equal(torch.isnan(f), at) and (f[:2][~at[:2]] == 448).all() and not f[2:][~at[2:]].any()
    assert torch.equal(scale, torch.tensor([1 / 448, 1 / 448, INF, INF], device=dev))
    w = torch.ones(40, device=dev)
    for res in (None, torch.zeros_like(x)):
        q, scale = ssm_scan.rms_norm_8bit(x, w, residual=res)[:2]
        f = q.float()
        assert (f[0] == 448).all() and torch.isnan(f[[1, 3]]).all()                # a NaN is its row's
        assert torch.equal(torch.isnan(f[2]), at[2]) and not f[2][~at[2]].any()    # the rest of an infinity's row is zeros
        assert (scale[1:] == 1).all()


@pytest.mark.parametrize("rows", [16, 128])   # the kernel for few rows, tiles
def test_products_are_added_eight_at_a_time(dev, rows):
    """2^16 at place 0 and -2^16 at place 127 leave what a product at place p adds: 2^3 is kept everywhere; what is below 2^-13 of
    the largest of its eight (places 0..7, 120..127) is lost there, and there alone."""
    p = torch.arange(1, 127)
    for e, kept in ((3, torch.ones(126, dtype=torch.bool)), (2, (p > 7) & (p < 120)), (-2, (p > 7) & (p < 120))):
        x, w = torch.zeros(128, 128), torch.full((16, 128), 2.0 ** (e // 2))
        x[:, 0] = x[:, 127] = 256.0
        w[:, 0], w[:, 127] = 256.0, -256.0
        x[p, p] = 2.0 ** (e - e // 2)
        ones = torch.ones(128, device=dev)
        y = torch.cat([ssm_scan.linear_8bit(t.to(F8).to(dev), ones[:rows], w.to(F8).to(dev), ones[:16], dtype=torch.float16) for t in x.split(rows)])
        assert torch.equal(y[1:127, 0].cpu() == 2.0 ** e, kept) and not y[1:127, 0].cpu()[~kept].any()
