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


@pytest.mark.parametrize("H", [16, 272, 512, 1024, 2048, 4096, 8192, 16384])
@pytest.mark.parametrize("stream", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_rows_of_zeros_and_rows_whose_squares_overflow(ops, H, stream, eps):
    """Zeros have a scale of 1 without an epsilon, too; squares beyond fp32 a NaN one.  Ordinary rows between them are
    what they are alone."""
    import test_gpu_norm_fp8 as norm
    x, w, r = norm._case(7, H, stream, seed=H)
    for row, by in ((1, 0.0), (3, 2.0 ** 90), (4, 0.0), (5, -(2.0 ** 90))):
        x[row] *= by
        if r is not None:
            r[row] *= by
    x[1, ::2] = -0.0
    run = lambda rows, unit: ops.add_rmsnorm_fp8(x[rows].cuda(), w.cuda(), eps, None if r is None else r[rows].cuda(), unit_offset=unit)
    for unit in (False, True):
        q, scale, _ = run(list(range(7)), unit)
        for row in (1, 4):
            assert (q[row].float() == 0).all() and scale[row] == 1
        assert torch.isnan(scale[[3, 5]]).all()
        for row in (0, 2, 6):
            alone = run([row], unit)
            assert torch.equal(alone[0].view(torch.uint8)[0], q.view(torch.uint8)[row]) and alone[1][0] == scale[row]
        norm._check([v if v is None else v[[0, 2, 6]] for v in run(list(range(7)), unit)], x[[0, 2, 6]], w,
                    r if r is None else r[[0, 2, 6]], unit, eps)
