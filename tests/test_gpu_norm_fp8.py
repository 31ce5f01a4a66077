"""Residual add + RMSNorm to e4m3 (ops.add_rmsnorm_fp8) against 64 bits.

Tolerances, derived: the stream s is one rounding of an fp32 sum, so it is equal.  The fp32 sum of
squares of H <= 16384 positive terms is at most 32 terms deep in a thread and 5 + 16 levels across
threads: 53 roundings of 2^-24, halved by the square root; the rsqrt, its argument, two products,
a reciprocal and a division add under 12 more.  So y and the scale are within 64 * 2^-24 relative, and
q within half an e4m3 step (2^-4 of the value, 2^-10 below the normals) of y / scale, widened by twice that."""

import pytest
import torch

from oracle import chunk as ref

pytestmark = pytest.mark.gpu
REL = 64 * 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


def _case(T, H, stream, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).mul(spread).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(torch.bfloat16)
    r = None if stream is None else (torch.randn(T, H, generator=g) * 3 * spread).to(stream)
    return x, w, r


def _check(got, x, w, r, unit, eps=1e-6):
    q, scale, s = (None if v is None else v.cpu() for v in got)
    y, want, stream = ref.add_rmsnorm(x, w, eps, r, unit)
    if r is None:
        assert s is None
    else:
        assert s.dtype == r.dtype and torch.equal(s, stream)
    assert ((scale.double() - want).abs() <= REL * want).all()
    e = y / want[:, None]
    off = (q.float().double() - e).abs()
    half = torch.maximum(e.abs() * 2.0 ** -4, torch.full_like(e, 2.0 ** -10))
    assert (off <= half * (1 + 2 * REL) + 2 * REL * e.abs()).all()


@pytest.mark.parametrize("stream", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 16), (1, 8192), (3, 256), (9, 272), (17, 512), (5, 1024), (7, 1040), (2, 2048),
                                 (3, 4096), (2, 4112), (130, 5120), (2, 16384), (3, 10000)])
def test_against_64_bits(ops, T, H, stream):
    x, w, r = _case(T, H, stream, seed=T + H)
    unit = (T + H // 16) % 2 == 0
    _check(ops.add_rmsnorm_fp8(x.cuda(), w.cuda(), 1e-6, None if r is None else r.cuda(), unit_offset=unit), x, w, r, unit)


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
def test_strided_rows_and_in_place_stream(ops, stream):
    x, w, r = _case(6, 512, stream, seed=4)
    xs = torch.full((6, 640), 7.0, dtype=torch.bfloat16, device="cuda")
    rs = torch.full((6, 576), 5.0, dtype=stream, device="cuda")
    xs[:, 64:576] = x.cuda()
    rs[:, :512] = r.cuda()
    view = rs[:, :512]
    q, scale, s = ops.add_rmsnorm_fp8(xs[:, 64:576], w.cuda(), 1e-6, view, residual_out=view)
    assert s.data_ptr() == rs.data_ptr()
    _check((q, scale, s.contiguous()), x, w, r, False)
    assert (rs[:, 512:] == 5.0).all()


def test_rows_of_zeros_infinities_and_nan(ops):
    x, w, _ = _case(5, 1024, None, seed=5)
    x[1] = 0
    x[2, 100] = float("inf")
    x[3, 7] = float("nan")
    q, scale, _ = ops.add_rmsnorm_fp8(x.cuda(), w.cuda(), 1e-6)
    q, scale = q.cpu().float(), scale.cpu()
    assert scale[1] == 1 and (q[1] == 0).all()
    # an infinity makes 1 / rms zero: its own element is inf * 0
    for row in (2, 3):
        assert not torch.isfinite(scale[row]) and not torch.isfinite(q[row] * scale[row]).any()
    keep = [0, 4]
    y, want, _ = ref.add_rmsnorm(x[keep], w, 1e-6)
    assert ((scale[keep].double() - want).abs() <= REL * want).all()


@pytest.mark.parametrize("spread", [2.0 ** -60, 2.0 ** 55])
def test_far_magnitudes(ops, spread):
    x, w, r = _case(3, 768, torch.float32, seed=6, spread=spread)
    eps = 0.0 if spread < 1 else 1e-6
    _check(ops.add_rmsnorm_fp8(x.cuda(), w.cuda(), eps, r.cuda()), x, w, r, False, eps)


def test_no_rows(ops):
    q, scale, s = ops.add_rmsnorm_fp8(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"),
                                      torch.ones(64, dtype=torch.bfloat16, device="cuda"), 1e-6,
                                      torch.empty(0, 64, device="cuda"))
    assert q.shape == s.shape == (0, 64) and scale.shape == (0,)


def test_refusals(ops):
    from okc_b200._lib import OkcError
    x, w, r = (v.cuda() for v in _case(2, 64, torch.float32))
    bad = [dict(x=x.float()), dict(w=w.float()), dict(w=w[:32]), dict(residual=r.half()), dict(residual=r[:1]),
           dict(x=x[:, :40], w=w[:40], residual=None), dict(residual=None, residual_out=r), dict(residual=r.cpu()),
           dict(residual_out=r.to(torch.bfloat16)), dict(x=x.t()), dict(x=x[:, 1:17], w=w[:16], residual=None)]
    for kw in bad:
        args = dict(x=x, w=w, residual=r)
        args.update(kw)
        with pytest.raises(OkcError):
            ops.add_rmsnorm_fp8(args.pop("x"), args.pop("w"), 1e-6, **args)
    wide = torch.zeros(1, 16400, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(OkcError):
        ops.add_rmsnorm_fp8(wide, wide[0], 1e-6)
