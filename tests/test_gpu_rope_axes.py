"""Multi-axis rotary append (ops.rope_axes_kv_append) against 64 bits.

Tolerances, derived: the reduced angle is rounded to fp32 (2^-24 * pi), its sine and cosine to 2 units and the
rotation takes 3 fp32 roundings: under 2^-20 (|a| + |b|) of the pair's values.  q is rounded to
bf16 (2^-8 relative), k and v after an fp32 division to e4m3 (2^-4, 2^-10 below the normals)."""

import pytest
import torch

from oracle import chunk as ref

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


def _case(new, old, Hq, Hkv, D, P, R, axes, far=0, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    B, T = len(new), sum(new) + pad
    full = [a + b for a, b in zip(new, old)]
    width = max(-(-f // P) for f in full) + 1
    pool = B * width + 2
    table = torch.randperm(pool, generator=g)[:B * width].to(torch.int32).view(B, width)
    c = {"qkv": torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16),
         "positions": torch.randint(0, 200, (max(axes) + 1, T), generator=g) + far,
         "axes": axes, "inv_freq": 1.0 / (5e5 ** (torch.arange(R).float() / R)),
         "cu_q": torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32),
         "seq_lens": torch.tensor(full, dtype=torch.int32), "page_table": table,
         "k_cache": torch.randint(0, 120, (pool, P, Hkv, D), generator=g).to(torch.uint8).view(E4M3),
         "v_cache": torch.randint(0, 120, (pool, P, Hkv, D), generator=g).to(torch.uint8).view(E4M3),
         "k_scale": 0.01 + 0.05 * torch.rand(Hkv, generator=g), "v_scale": 0.01 + 0.05 * torch.rand(Hkv, generator=g)}
    return c


def _cuda(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def _run_and_check(ops, c, Hq, Hkv, D, half):
    d = _cuda(c)
    T, R = c["qkv"].shape[0], len(c["axes"])
    q = torch.full((T, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
    assert ops.rope_axes_kv_append(**d, Hq=Hq, Hkv=Hkv, D=D, half=half, q_out=q) is q
    assert ops.read_device_error("rope_axes") == 0
    out = ref.rope_axes(c["qkv"], c["positions"], c["axes"], c["inv_freq"], Hq, Hkv, D, half)
    x = c["qkv"].double().view(T, Hq + 2 * Hkv, D).abs()
    size = torch.zeros_like(x)  # |a| + |b| of each element's pair
    for i in range(R):
        u, v = (i, i + R) if half else (2 * i, 2 * i + 1)
        size[..., u] = size[..., v] = x[..., u] + x[..., v]
    slack = 2.0 ** -20 * size
    places = ref.places(c["cu_q"], c["seq_lens"])
    n = len(places)
    q = q.cpu()
    assert (q[n:] == 3.0).all()
    assert ((q[:n].double() - out[:n, :Hq]).abs() <= 2.0 ** -8 * out[:n, :Hq].abs() + slack[:n, :Hq] * 1.01).all()
    P = c["k_cache"].shape[1]
    for name, first in (("k", Hq), ("v", Hq + Hkv)):
        got, before = d[name + "_cache"].cpu(), c[name + "_cache"]
        scale = c[name + "_scale"].double()[:, None]
        touched = torch.zeros(got.shape[:2], dtype=torch.bool)
        for t, (b, p) in enumerate(places):
            page = int(c["page_table"][b, p // P])
            touched[page, p % P] = True
            e = out[t, first:first + Hkv] / scale
            tol = torch.maximum(e.abs() * 2.0 ** -4, torch.full_like(e, 2.0 ** -10)) + 1.01 * (
                slack[t, first:first + Hkv] / scale) + 2.0 ** -23 * e.abs()
            assert ((got[page, p % P].float().double() - e).abs() <= tol).all()
        assert torch.equal(got.view(torch.uint8)[~touched], before.view(torch.uint8)[~touched])


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("new,old,Hq,Hkv,D,P,R,far", [
    ([1], [0], 4, 1, 64, 1, 32, 0), ([1, 1, 1], [9, 0, 31], 8, 8, 128, 16, 64, 0), ([5, 0, 17], [3, 8, 0], 7, 1, 128, 16, 48, 1000000),
    ([40], [100], 6, 2, 64, 64, 16, 50000), ([3, 2], [20, 5], 2, 1, 256, 7, 128, 0), ([2], [2], 3, 3, 8 * 5, 16, 8, 17),
    ([1] * 70, [4] * 70, 2, 2, 64, 16, 32, 0)])
def test_against_64_bits(ops, new, old, Hq, Hkv, D, P, R, far, half):
    for axes in (ops.rope_sections((R // 4, R - R // 4)), tuple(i % 3 for i in range(R))):
        c = _case(new, old, Hq, Hkv, D, P, R, axes, far, seed=R + P, pad=2)
        _run_and_check(ops, c, Hq, Hkv, D, half)


def test_one_axis_equals_the_decode_append(ops):
    """With one axis at the cache positions and interleaved pairs this is rope_kv_append, but for the
    angle, which that operator forms in fp32 (its positions are small here, so that both agree closely)."""
    Hq, Hkv, D, P, B = 8, 2, 128, 16, 5
    c = _cuda(_case([1] * B, [3, 0, 15, 16, 40], Hq, Hkv, D, P, D // 2, (0,) * (D // 2), seed=8))
    pos = c["seq_lens"].long() - 1
    c["positions"] = pos[None].contiguous()
    kc, vc = c["k_cache"].clone(), c["v_cache"].clone()
    q = ops.rope_axes_kv_append(**c, Hq=Hq, Hkv=Hkv, D=D)
    q2 = ops.rope_kv_append(c["qkv"], pos, c["page_table"], kc, vc, c["k_scale"], c["v_scale"], Hq, Hkv, D, c["inv_freq"])
    # fp32 angles below 41: off by 2^-24 * 41, in all under 2^-8 of a value plus 2^-17 of the pair
    assert ((q.float() - q2.float()).abs() <= 2.0 ** -7 * q2.float().abs() + 2.0 ** -15).all()
    assert torch.equal(c["v_cache"].view(torch.uint8), vc.view(torch.uint8))


def test_positions_off_the_table_are_skipped(ops):
    Hq, Hkv, D, P = 2, 1, 64, 16
    c = _case([2, 2, 2], [30, 5, 5], Hq, Hkv, D, P, 32, (0,) * 32, seed=3)
    c["seq_lens"][0] = 1000   # past the table's columns
    c["seq_lens"][1] = 1      # the first of two rows before position 0
    c["page_table"][2, 0] = 10 ** 6
    d = _cuda(c)
    q = ops.rope_axes_kv_append(**d, Hq=Hq, Hkv=Hkv, D=D)
    from okc_b200 import _lib
    assert ops.read_device_error("rope_axes") == _lib.DEVERR_PAGE and ops.read_device_error("rope_axes") == 0
    changed = (d["k_cache"].cpu().view(torch.uint8) != c["k_cache"].view(torch.uint8)).any(-1).any(-1)
    want = torch.zeros_like(changed)
    want[int(c["page_table"][1, 0]), 0] = True
    assert torch.equal(changed, want)
    assert torch.isfinite(q.float()).all()


def test_refusals(ops):
    from okc_b200._lib import OkcError
    c = _cuda(_case([2], [3], 2, 1, 64, 16, 32, (0, 1) * 16, seed=1))
    kw = dict(Hq=2, Hkv=1, D=64)
    bad = [dict(axes=(0,) * 31), dict(axes=(0,) * 12, inv_freq=c["inv_freq"][:12].contiguous()), dict(axes=(2,) * 32), dict(axes=(5,) * 32),
           dict(positions=c["positions"].int()), dict(positions=c["positions"][:, :1]), dict(qkv=c["qkv"].float()),
           dict(cu_q=c["cu_q"].long()), dict(cu_q=c["cu_q"][:1]), dict(seq_lens=c["seq_lens"].cpu()), dict(Hq=3),
           dict(k_cache=c["k_cache"].view(torch.uint8)), dict(v_cache=c["v_cache"][:1]), dict(k_scale=c["k_scale"].double()),
           dict(page_table=c["page_table"].long()), dict(axes=(0,) * 40, inv_freq=torch.ones(40, device="cuda"))]
    for more in bad:
        with pytest.raises(OkcError):
            ops.rope_axes_kv_append(**{**c, **kw, **more})
