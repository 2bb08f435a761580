"""The linear layer at the ends of its range: rows whose tiles pass 32-bit offsets, arguments of the activation beyond the
operands' type, operands whose rows share their memory, scales whose product leaves float32, GELU's tail, operands of one
channel with any stride."""

import pytest
import torch

import ssm_scan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("MN,K", [(3331, 4300000), (1800, 8500000)])
def test_long_rows(dev, MN, K):
    """Row 255 (or 127) of a tile begins more than 2^31 bytes after its first.  Small whole numbers at both ends of the rows:
    sums are exact."""
    if torch.cuda.mem_get_info()[0] < 5 * MN * K:
        pytest.skip("not enough memory")
    r = torch.Generator().manual_seed(1)
    cols = torch.cat([torch.arange(64), torch.arange(K - 64, K)]).to(dev)
    x, w = (torch.zeros(MN, K, dtype=BF16, device=dev) for _ in range(2))
    small = [torch.randint(-2, 3, (MN, 128), generator=r).to(dev).float() for _ in range(2)]
    for t, s in zip((x, w), small):
        t[:, :64] = s[:, :64].to(BF16)
        t[:, -64:] = s[:, 64:].to(BF16)
    y = ssm_scan.linear_act(x, w)
    assert len(cols) == 128 and torch.equal(y, (small[0] @ small[1].t()).to(BF16))
    del x, w, t
    torch.cuda.empty_cache()
