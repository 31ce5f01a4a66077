"""Residual add + RMSNorm to e4m3 (ops.add_rmsnorm_fp8) where one rounding decides: quotients on the border of two e4m3
values, rows of zeros without an epsilon."""

import pytest
import torch

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


@pytest.mark.parametrize("H", [512, 1024, 4096, 16384])
def test_quotients_are_those_of_a_division(ops, H):
    """Rows of +-1 have a root mean square of 1, so that y is the weight: every weight of 256 steps an octave below each
    of 128 largest ones, among them many that lie on a tie of two e4m3 values, which a product with the reciprocal misses
    (4.75 / 448 and 0.890625, for one).  Equal, bit for bit."""
    g = torch.Generator().manual_seed(H)
    sign = torch.where(torch.rand(2, H, generator=g) < 0.5, -1.0, 1.0).to(torch.bfloat16)
    vals = torch.arange(0x3F00, 0x4400, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # 0.5 to 512
    ties = 0
    for top in range(128):
        for factor in (2.0 ** -7, 4.0, 2.0 ** 6):
            most = torch.tensor((128 + top) / 128).mul(factor)
            below = vals[vals.float() <= most] if factor > 1 else (vals.float() * 2.0 ** -9).to(torch.bfloat16)
            below = below[below.float() <= most]
            w = below[torch.randint(0, len(below), (H,), generator=g)]
            w[H // 3] = most.to(torch.bfloat16)
            q, scale, _ = ops.add_rmsnorm_fp8(sign.cuda(), w.cuda(), 0.0)
            want = (most / 448).float()
            assert (scale.cpu() == want).all()
            y = sign.float() * w.float()
            expect = (y / want).to(E4M3)
            ties += int(((y / want).to(E4M3).float() != (y * (1 / want)).to(E4M3).float()).sum())
            assert torch.equal(q.cpu().view(torch.uint8), expect.view(torch.uint8))
    assert ties > 0
