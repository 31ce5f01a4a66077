"""Projection with an epilogue (ops.linear) where its last steps decide: activations of fp32 outputs."""

import math

import pytest
import torch

from oracle import chunk as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


@pytest.mark.parametrize("M", [16, 100, 400])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activations_of_fp32_outputs(ops, M, act):
    """Every row of x picks one column of w, so that the activation's argument is exact: every bf16 from 2^-12 to 64
    of both signs.  The exponential is within 2^-22 (ex2.approx) and a rounding, the addition rounds once, the division is
    within 2^-22 (__fdividef): 2^-21 + 2^-23 of the result.  The tanh form's argument u of the exponential has five
    roundings, each of which the exponential multiplies by |u|, and where that passes 2^126 (the division's end) the
    result, below |v| 2^-126, is zero; the erf is within two units of 1, of which v takes a half."""
    vals = torch.arange(0x3980, 0x4280, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    vals = torch.cat([vals, -vals, torch.zeros(16 - 2 * len(vals) % 16, dtype=torch.bfloat16)])
    w = vals.view(-1, 16)
    x = torch.eye(16, dtype=torch.bfloat16).repeat(M // 16 + 1, 1)[:M]
    y = ops.linear(x.cuda(), w.cuda().contiguous(), act=act, out_dtype=torch.float32).cpu().double()
    v = w.double()[:, torch.arange(M) % 16].t()
    want = ref.act64(v, act)
    tol = torch.zeros_like(v)
    if act == "silu":
        tol = (2.0 ** -21 + 2.0 ** -23) * want.abs()
    elif act == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3).abs()
        want = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))  # without the 1 + tanh that cancels
        tol = (2.0 ** -21 + 2.0 ** -23 + 5 * 2.0 ** -24 * u) * want.abs() + 2.0 ** -126 * v.abs()
    elif act == "gelu":
        tol = 2.0 ** -22 * v.abs()
    off = (y - want).abs()
    assert (off <= tol).all(), f"off by {float((off / tol.clamp(min=1e-300)).max()):.1f} tolerances at {float(v.flatten()[(off / tol.clamp(min=1e-300)).argmax()])}"


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("M", [1, 17, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 16), (2, 32), (7, 1040), (31, 16), (33, 272)])
def test_the_narrowest_outputs(ops, M, N, K, dtype):
    import test_gpu_linear as lin
    c = lin._case(M, N, K, dtype, seed=M + N, residual=torch.float32)
    for out in (torch.float32, torch.bfloat16):
        lin._check(ops.linear(**lin._cuda(c), act="silu", out_dtype=out), c, "silu", f"{M} {N} {K} {out}")
