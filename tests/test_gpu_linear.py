"""Projection with an epilogue (ops.linear) against 64 bits.

Tolerance, derived: products of e4m3 or bf16 values are exact in fp32.  An output takes K / 16 or
K / 32 MMA steps and up to 8 split sums; each addition may lose one unit (2^-23) of a partial sum that
is at most a = sum |x||w|, and a step aligns its products to the largest with the same loss: under
(K / 8 + 16) * 2^-23 * a.  Scales and bias add 3 roundings of 2^-24 of their results.  Every
activation here has a slope of at most 1.13 and is computed within 2^-20 of max(|y|, 1) (one
exponential of an argument below 88, whose error grows with it by 2^-24 per unit, where the result is not yet 0 or y).  The
output is rounded once."""

import pytest
import torch

from oracle import chunk as ref

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


def _case(M, N, K, dtype, seed=0, scales=True, bias=True, residual=None):
    g = torch.Generator().manual_seed(seed)
    c = {}
    if dtype == "e4m3":
        c["x"] = (torch.randn(M, K, generator=g) * 90).clamp(-448, 448).to(E4M3)
        c["w"] = (torch.randn(N, K, generator=g) * 90).clamp(-448, 448).to(E4M3)
    else:
        c["x"] = (torch.randn(M, K, generator=g) * 90).to(torch.bfloat16)
        c["w"] = (torch.randn(N, K, generator=g) * 90).to(torch.bfloat16)
    if scales:
        c["x_scale"] = (0.5 + torch.rand(M, generator=g)) / 90
        c["w_scale"] = (0.5 + torch.rand(N, generator=g)) / (90 * K ** 0.5)
    if bias:
        c["bias"] = torch.randn(N, generator=g).to(torch.bfloat16)
    if residual is not None:
        c["residual"] = torch.randn(M, N, generator=g).to(residual)
    return c


def _cuda(c):
    return {k: v.cuda() for k, v in c.items()}


def _check(y, c, act, what=""):
    K = c["x"].shape[1]
    want, a = ref.linear(act=act, **c)
    y = y.cpu()
    pre = (K / 8 + 16) * 2.0 ** -23 * a + 3 * 2.0 ** -24 * (a + 1)
    tol = 1.13 * pre + 2.0 ** -20 * want.abs().clamp(min=1) + torch.finfo(y.dtype).eps / 2 * want.abs()
    off = (y.double() - want).abs()
    assert (off <= tol).all(), f"{what}: off by up to {(off / tol).max():.2f} tolerances at {int((off / tol).argmax())}"


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (1, 8192, 1024), (2, 1, 16), (3, 130, 48), (5, 257, 4112), (8, 1000, 512),
                                   (16, 384, 2064), (17, 129, 640), (33, 515, 1024), (64, 1280, 256), (65, 200, 8192),
                                   (100, 4099, 272), (128, 512, 1040), (129, 255, 512), (200, 1025, 144),
                                   (256, 256, 4096), (257, 700, 1296), (515, 300, 384), (777, 1283, 1040), (1025, 512, 64)])
def test_shapes(ops, M, N, K, dtype):
    c = _case(M, N, K, dtype, seed=M + N + K)
    _check(ops.linear(**_cuda(c), out_dtype=torch.float32), c, None, f"{M} {N} {K} fp32")
    _check(ops.linear(**_cuda(c)), c, None, f"{M} {N} {K} bf16")


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("residual", [torch.bfloat16, torch.float32])
def test_epilogues(ops, M, act, residual):
    c = _case(M, 333, 320, "e4m3", seed=M, residual=residual)
    for out in (torch.bfloat16, torch.float32):
        _check(ops.linear(**_cuda(c), act=act, out_dtype=out), c, act, f"{M} {act} {residual} {out}")


@pytest.mark.parametrize("M", [4, 150])
def test_parts_left_out(ops, M):
    for scales in (False, True):
        for bias in (False, True):
            c = _case(M, 96, 160, "bf16", seed=1, scales=scales, bias=bias)
            c["x"], c["w"] = c["x"] / 90, c["w"] / 90
            _check(ops.linear(**_cuda(c)), c, None)
    c = _case(M, 96, 160, "e4m3", seed=2)
    c["w_scale"] = c["w_scale"][:1]
    _check(ops.linear(**_cuda(c)), c, None)
    del c["x_scale"]
    _check(ops.linear(**_cuda(c)), c, None)


@pytest.mark.parametrize("M,N", [(7, 250), (300, 250), (300, 256)])
def test_strides_and_in_place_residual(ops, M, N):
    c = _case(M, N, 256, "e4m3", seed=3, residual=torch.float32)
    d = _cuda(c)
    xs = torch.zeros(M, 400, dtype=torch.uint8, device="cuda")
    ws = torch.zeros(N, 272, dtype=torch.uint8, device="cuda")
    xs[:, 16:272] = d["x"].view(torch.uint8)
    ws[:, :256] = d["w"].view(torch.uint8)
    d["x"], d["w"] = xs.view(E4M3)[:, 16:272], ws.view(E4M3)[:, :256]
    r = torch.full((M, N + 3), 9.0, device="cuda")
    r[:, :N] = d["residual"]
    d["residual"] = r[:, :N]
    y = ops.linear(**d, act="silu", out=r[:, :N])
    assert y.data_ptr() == r.data_ptr()
    _check(y.contiguous(), c, "silu")
    assert (r[:, N:] == 9.0).all()


def test_nonfinite_operands_stay_in_their_rows(ops):
    for M in (6, 200):
        c = _case(M, 140, 192, "e4m3", seed=7)
        d = _cuda(c)
        d["x"].view(torch.uint8)[2, 100] = 0x7F  # NaN
        d["x_scale"][4] = float("inf")
        for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
            y = ops.linear(**d, act=act).float().cpu()
            assert torch.isnan(y[2]).all()
            # an infinite scale times the row's products: infinite where they are positive, whatever the bias
            assert not torch.isfinite(y[4][ref.linear(c["x"], c["w"])[0][4] > 0]).any()
            keep = [i for i in range(M) if i not in (2, 4)]
            assert torch.isfinite(y[keep]).all()


def test_equal_twice(ops):
    for M in (1, 30, 128, 300):
        d = _cuda(_case(M, 2048, 4096, "e4m3", seed=9))
        assert torch.equal(ops.linear(**d), ops.linear(**d))


def test_many_rows(ops):
    """More token rows than one pass of the grid's tiles, every one checked against fp32 products."""
    c = _cuda(_case(5000, 1500, 128, "e4m3", seed=11))
    y = ops.linear(**c, out_dtype=torch.float32)
    x, w = c["x"].float(), c["w"].float()
    want = x @ w.t() * c["x_scale"][:, None] * c["w_scale"] + c["bias"].float()
    a = x.abs() @ w.abs().t() * c["x_scale"][:, None] * c["w_scale"]
    # both sides in fp32: twice the accumulation's bound
    assert ((y - want).abs() <= 2 * (128 / 8 + 16) * 2.0 ** -23 * a + 8 * 2.0 ** -24 * (a + 4)).all()


def test_no_rows(ops):
    d = _cuda(_case(2, 64, 64, "e4m3"))
    d["x"], d["x_scale"] = d["x"][:0], d["x_scale"][:0]
    assert ops.linear(**d).shape == (0, 64)


def test_refusals(ops):
    from okc_b200._lib import OkcError
    d = _cuda(_case(4, 64, 64, "e4m3", residual=torch.float32))
    bf = _cuda(_case(4, 64, 64, "bf16"))
    bad = [dict(x=bf["x"]), dict(w=bf["w"]), dict(act="tanh"), dict(bias=d["bias"].float()), dict(bias=d["bias"][:1]),
           dict(x_scale=d["x_scale"].double()), dict(x_scale=d["x_scale"][:1]), dict(w_scale=d["w_scale"][:3]),
           dict(residual=d["residual"][:, :3]), dict(residual=d["residual"].half()), dict(out_dtype=torch.float16),
           dict(x=d["x"][:, :40], w=d["w"][:, :40]), dict(x=d["x"][:, :32]), dict(x=d["x"].t()), dict(x=d["x"].cpu()),
           dict(x=d["x"].float(), w=d["w"].float()), dict(bias=d["bias"].cpu()), dict(x=d["x"][:, 8:56], w=d["w"][:, 8:56]),
           dict(out=torch.empty(4, 64, device="cuda", dtype=torch.float16)), dict(out=torch.empty(64, 4, device="cuda").t())]
    for kw in bad:
        with pytest.raises(OkcError):
            ops.linear(**{**d, **kw})


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_tall_blocks_without_a_residual(ops, act, dtype):
    """bf16 outputs whose rows take 16-byte accesses, and the same products into rows that do not: equal."""
    c = _case(300, 352, 272, dtype, seed=31)
    d = _cuda(c)
    y = ops.linear(**d, act=act)
    _check(y, c, act)
    for cols, first in ((360, 8), (355, 0), (360, 3)):
        wide = torch.full((300, cols), 7.0, dtype=torch.bfloat16, device="cuda")
        out = wide[:, first:first + 352]
        assert torch.equal(ops.linear(**d, act=act, out=out), y)
        assert (wide[:, :first] == 7).all() and (wide[:, first + 352:] == 7).all()
