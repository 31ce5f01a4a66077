"""Ragged chunk attention over the paged e4m3 cache (ops.attn_chunk) against 64 bits.

Tolerance, derived: q.k is a sum of D <= 128 exact products in fp32, off by at most (D / 8) * 2^-23 of
sum |q||k|; with |q| ~ 2, |k| ~ 1, D = 128 that is below 2^-11 of a score unit after the softmax scale, and the
factors add 2^-22 of a score of at most 50, the cap's tanh (within 1.2e-6) 2^-14 at a cap of 50.  So each p is
within 2^-10.5 relative, plus its own rounding to f16 (2^-11, or 2^-25 of the row's largest p for the small ones): o is within 2^-9.5 of
a = sum p|v| before, and 2^-8 of itself by, the rounding to bf16."""

import math

import pytest
import torch

from oracle import chunk as ref

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


def _case(new, old, Hq, Hkv, D, P, seed=0, pad=0, cap=0.0, slopes=False, window=0, prefix=False, docs=False):
    g = torch.Generator().manual_seed(seed)
    B, T = len(new), sum(new) + pad
    full = [a + b for a, b in zip(new, old)]
    width = max(1, max(-(-f // P) for f in full)) + 1
    pool = B * width + 2
    c = {"q": (torch.randn(T, Hq, D, generator=g) * 2).to(torch.bfloat16),
         "page_table": torch.randperm(pool, generator=g)[:B * width].to(torch.int32).view(B, width),
         "cu_q": torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32),
         "seq_lens": torch.tensor(full, dtype=torch.int32), "sm_scale": 1 / math.sqrt(D), "softcap": cap, "window": window}
    for n in ("k", "v"):
        s = 0.01 + 0.02 * torch.rand(Hkv, generator=g)
        x = torch.randn(pool, P, Hkv, D, generator=g) / s[:, None]
        c[n + "_scale"], c[n + "_cache"] = s, x.clamp(-448, 448).to(E4M3)
    if slopes:
        c["slopes"] = 2.0 ** (-8.0 * (torch.arange(Hq) + 1).float() / Hq)
    if prefix:
        c["prefix_lens"] = torch.tensor([int(torch.randint(0, f + 3, (1,), generator=g)) for f in full], dtype=torch.int32)
    if docs:
        first = []
        for n, f in zip(new, full):
            at, start = f - n, 0
            for p in range(f - n, f):
                if int(torch.randint(0, 4, (1,), generator=g)) == 0:
                    start = p + int(torch.randint(0, 2, (1,), generator=g)) * 5  # some rows see nothing
                first.append(start)
        c["doc_start"] = torch.tensor(first + [0] * pad, dtype=torch.int32)
    return c


WIDE = False


@pytest.fixture(autouse=True, params=[False, True], ids=["narrow", "wide"])
def table_width(request):
    """Page tables as wide as the longest request, or with 4096 columns more (which no request reaches): few tiles
    and a narrow table let the short chunks' kernel take long chunks too, a wide one leaves them to the other."""
    global WIDE
    WIDE = request.param
    yield
    WIDE = False


def _cuda(c):
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    if WIDE:
        d["page_table"] = torch.nn.functional.pad(d["page_table"], (0, 4096), value=-1)
    return d


def _close(o, c, what=""):
    want, a = ref.attn_chunk(**c)
    n = want.shape[0]
    off = (o[:n].cpu().double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -9.5 * a
    assert (off <= tol).all(), f"{what}: off by up to {float((off / tol.clamp(min=1e-30)).max()):.2f} tolerances"


def _check(ops, c, what="", **more):
    T, Hq, D = c["q"].shape
    out = torch.full((T, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
    assert ops.attn_chunk(**_cuda(c), out=out, **more) is out
    assert ops.read_device_error("attn_chunk") == 0
    _close(out, c, what)
    assert (out[int(c["cu_q"][-1]):] == 3.0).all()


HEADS = [(4, 1, 64, 1), (16, 2, 64, 16), (8, 8, 128, 16), (7, 1, 128, 16), (64, 8, 128, 16), (16, 1, 128, 64), (20, 4, 64, 7),
         (32, 16, 64, 16), (24, 12, 64, 16)]


@pytest.mark.parametrize("Hq,Hkv,D,P", HEADS)
@pytest.mark.parametrize("kind", [dict(), dict(cap=20.0, slopes=True), dict(window=37), dict(cap=50.0, window=130)])
def test_decode(ops, Hq, Hkv, D, P, kind):
    c = _case([1, 1, 1, 1, 1], [0, 1, 31, 300, 77], Hq, Hkv, D, P, seed=Hq + D, pad=1, **kind)
    _check(ops, c, max_q=1)
    _check(ops, c)


@pytest.mark.parametrize("Hq,Hkv,D,P", HEADS)
@pytest.mark.parametrize("kind", [dict(), dict(cap=30.0, slopes=True, docs=True), dict(window=21, prefix=True),
                                  dict(prefix=True, docs=True, slopes=True), dict(cap=50.0, prefix=True)])
def test_chunks(ops, Hq, Hkv, D, P, kind):
    c = _case([3, 0, 40, 1, 9], [50, 7, 0, 129, 2], Hq, Hkv, D, P, seed=Hq * D + P, pad=3, **kind)
    _check(ops, c, max_q=40)
    _check(ops, c)


@pytest.mark.parametrize("new,old", [([150], [200]), ([129, 257], [0, 63]), ([300, 1, 64], [5, 700, 130])])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (6, 2, 64), (5, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("kind", [dict(), dict(cap=30.0, slopes=True), dict(window=100, docs=True), dict(prefix=True, cap=20.0, docs=True)])
def test_long_chunks(ops, new, old, Hq, Hkv, D, kind):
    c = _case(new, old, Hq, Hkv, D, 16, seed=sum(new) + Hq, **kind)
    _check(ops, c, max_q=max(new))


def test_long_context_split_over_the_grid(ops):
    c = _case([1, 2], [9000, 4500], 8, 2, 128, 16, seed=1, cap=30.0)
    _check(ops, c, max_q=2)
    c = _case([1], [20000], 4, 1, 64, 1, seed=2, slopes=True)
    _check(ops, c, max_q=1)
    c = _case([33], [6000], 4, 1, 64, 16, seed=2)
    _check(ops, c, max_q=33)


def test_large_scores(ops):
    """Scores of hundreds: capped at 50, or a softmax that is one key's."""
    for cap in (0.0, 50.0):
        c = _case([2, 70], [100, 40], 8, 2, 128, 16, seed=4, cap=cap)
        c["sm_scale"] = 1.0
        o = ops.attn_chunk(**_cuda(c), max_q=70).cpu().double()
        want, a = ref.attn_chunk(**c)
        # a score of up to 350 is off by 2^-23 * (16 * sum |q||k| + 350 * 4): under 2^-8.5 for sums up to 1500
        assert ((o - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * a).all()


def test_far_query_magnitudes(ops):
    c = _case([2, 66], [60, 9], 8, 2, 64, 16, seed=5)
    c["q"][:, 0] *= 2.0 ** -40
    c["q"][:, 1] *= 2.0 ** 30
    c["sm_scale"] /= 4
    d = _cuda(c)
    o = ops.attn_chunk(**d, max_q=66).cpu()
    c["q"][:, 1] = 0  # heads apart: compare all but the huge one, which is one key's value
    want, a = ref.attn_chunk(**c)
    keep = [0, 2, 3, 4, 5, 6, 7]
    assert ((o.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9.5 * a)[:, keep].all()
    assert torch.isfinite(o.float()).all()


@pytest.mark.parametrize("new,old", [([4, 1], [20, 33]), ([140], [10])])
def test_nan_outside_a_rows_interval_does_not_reach_it(ops, new, old):
    """Pages hold NaN past the sequence, before the window and at later tokens of the chunk."""
    c = _case(new, old, 8, 2, 128, 16, seed=6, window=12)
    clean = _cuda(c)
    o = ops.attn_chunk(**clean, max_q=max(new))
    bad = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in clean.items()}
    last = []
    for b in range(len(new)):
        full, n = int(c["seq_lens"][b]), new[b]
        width = c["page_table"].shape[1] * 16
        for p in list(range(full, width)) + list(range(0, max(0, full - n + 1 - 12))) + [full - 1]:
            page = int(c["page_table"][b, p // 16])
            for t in ("k_cache", "v_cache"):
                bad[t].view(torch.uint8)[page, p % 16] = 0x7F if p % 2 else 0xFF
        last.append(int(c["cu_q"][b + 1]) - 1)
    o2 = ops.attn_chunk(**bad, max_q=max(new))
    keep = [t for t in range(sum(new)) if t not in last]  # only the last token sees the last position
    assert torch.equal(o[keep], o2[keep])
    assert torch.isnan(o2[last].float()).all()


def test_a_visible_nan_value_stays_in_its_column(ops):
    for new, old in (([3], [40]), ([130], [40])):
        c = _case(new, old, 4, 2, 64, 16, seed=7)
        d = _cuda(c)
        o = ops.attn_chunk(**d, max_q=max(new))
        d["v_cache"].view(torch.uint8)[int(c["page_table"][0, 2]), 9, 1, 5] = 0x7F  # position 41: the second new token
        o2 = ops.attn_chunk(**d, max_q=max(new)).float()
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[1:, 2:, 5] = True
        assert torch.equal(torch.isnan(o2), hit)
        assert torch.equal(o2[~hit], o.float()[~hit])


def test_rows_that_see_nothing_are_zero(ops):
    for n in (3, 90):
        c = _case([n, n], [10, 0], 8, 2, 64, 16, seed=8)
        c["doc_start"] = torch.full((2 * n,), 10 ** 6, dtype=torch.int32)
        c["doc_start"][n:] = 0
        _check(ops, c, max_q=n)
        c["seq_lens"][1] = 0  # rows before position 0
        o = ops.attn_chunk(**_cuda(c), max_q=n)
        assert (o == 0).all()


def test_bad_pages_read_zeros_and_set_the_error(ops):
    from okc_b200 import _lib
    for n in (2, 100):
        c = _case([n], [40], 8, 2, 64, 16, seed=9)
        zero = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        page = int(c["page_table"][0, 1])
        zero["k_cache"].view(torch.uint8)[page] = 0
        zero["v_cache"].view(torch.uint8)[page] = 0
        for bad in (-1, 10 ** 6):
            c["page_table"][0, 1] = bad
            o = ops.attn_chunk(**_cuda(c), max_q=n)
            assert ops.read_device_error("attn_chunk") == _lib.DEVERR_PAGE
            _close(o, zero)
        c["page_table"][0, 1] = page
        c["seq_lens"][0] = c["page_table"].shape[1] * 16 + 30  # past the table's columns
        ops.attn_chunk(**_cuda(c), max_q=n)
        assert ops.read_device_error("attn_chunk") == _lib.DEVERR_PAGE


def test_strided_rows(ops):
    for n in (1, 80):
        c = _case([n, 2], [33, 8], 8, 2, 128, 16, seed=10)
        d = _cuda(c)
        wide = torch.zeros(n + 2, 12, 128, dtype=torch.bfloat16, device="cuda")
        wide[:, 2:10] = d["q"]
        d["q"] = wide[:, 2:10]
        out = torch.full((n + 2, 10, 128), 5.0, dtype=torch.bfloat16, device="cuda")
        table = torch.full((2, d["page_table"].shape[1] + 3), -1, dtype=torch.int32, device="cuda")
        table[:, :-3] = d["page_table"]
        d["page_table"] = table[:, :-3]
        ops.attn_chunk(**d, max_q=n, out=out[:, 1:9])
        _close(out[:, 1:9], c)
        assert (out[:, 0] == 5).all() and (out[:, 9] == 5).all()


def test_equal_twice_and_whatever_max_q_says(ops):
    c = _cuda(_case([2, 150, 1], [300, 64, 2000], 8, 2, 128, 16, seed=11, cap=30.0))
    o = ops.attn_chunk(**c, max_q=150)
    assert torch.equal(o, ops.attn_chunk(**c, max_q=150))
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    for m in (None, 1, 10 ** 6):
        _close(ops.attn_chunk(**c, max_q=m), cpu)


def test_many_requests(ops):
    c = _case([1] * 700, [(7 * i) % 90 for i in range(700)], 4, 2, 64, 16, seed=12)
    _check(ops, c, max_q=1)
    d = _cuda(_case([1] * 2049, [1] * 2049, 4, 2, 64, 16, seed=12))
    from okc_b200._lib import OkcError
    with pytest.raises(OkcError):
        ops.attn_chunk(**d, max_q=1)


def test_decode_matches_the_decode_operator(ops):
    """Without cap, bias and masks one token a request is what attn_decode computes."""
    c = _cuda(_case([1] * 6, [5, 100, 33, 700, 64, 0], 16, 2, 64, 1, seed=13))
    o = ops.attn_chunk(**c, max_q=1)
    o2 = ops.attn_decode(c["q"], c["k_cache"], c["v_cache"], c["page_table"], c["seq_lens"], c["k_scale"], c["v_scale"], c["sm_scale"])
    torch.testing.assert_close(o.float(), o2.float(), rtol=2e-2, atol=2e-2)


def test_refusals(ops):
    from okc_b200._lib import OkcError
    c = _cuda(_case([2], [3], 4, 2, 64, 16, seed=1, slopes=True, prefix=True, docs=True))
    bad = [dict(q=c["q"].float()), dict(q=c["q"][:, :3]), dict(q=c["q"].transpose(0, 1)), dict(softcap=-1.0),
           dict(softcap=float("nan")), dict(sm_scale=float("inf")), dict(window=-1), dict(slopes=c["slopes"][:2]),
           dict(slopes=c["slopes"].double()), dict(prefix_lens=c["prefix_lens"].long()), dict(doc_start=c["doc_start"][:1]),
           dict(cu_q=c["cu_q"].cpu()), dict(page_table=c["page_table"][:, :0]), dict(k_cache=c["k_cache"][..., :32]),
           dict(v_cache=c["v_cache"].float()), dict(k_scale=c["k_scale"][:1]), dict(max_q=-1),
           dict(q=c["q"][..., :32].contiguous(), k_cache=c["k_cache"][..., :32].contiguous(), v_cache=c["v_cache"][..., :32].contiguous())]
    for kw in bad:
        with pytest.raises(OkcError):
            ops.attn_chunk(**{**c, **kw})


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("new,old,prefix", [([150, 40], [300, 10], [430, 50]), ([400], [100], [260]), ([70, 70, 70], [900, 0, 64], [0, 70, 1000]),
                                            ([2000], [100], [2100])])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (14, 2, 64)])
def test_a_bias_over_keys_on_both_sides(ops, new, old, prefix, cap, Hq, Hkv, D):
    """Rows inside a prefix that ends blocks behind them see keys ahead of their position, lowered as those behind are."""
    c = _case(new, old, Hq, Hkv, D, 16, seed=len(new) + Hq, cap=cap, slopes=True)
    c["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32)
    _check(ops, c, max_q=max(new))
    c["window"] = 90
    _check(ops, c, max_q=max(new))


@pytest.mark.parametrize("new", [1, 3])
def test_many_steps_of_64_wide_heads(ops, new):
    """Enough key steps for two blocks an SM, and a table that allows them where few are used."""
    B = 40
    c = _case([new] * B, [(331 * i) % 1900 + 300 for i in range(B)], 16, 8, 64, 16, seed=20, cap=30.0)
    _check(ops, c, max_q=new)
    c["seq_lens"] = torch.tensor([(5 * i) % 40 + new for i in range(B)], dtype=torch.int32)
    _check(ops, c, max_q=new)
    d = _cuda(c)
    assert torch.equal(ops.attn_chunk(**d, max_q=new), ops.attn_chunk(**d, max_q=new))


def test_one_request_with_rows_behind_it(ops):
    """A single request of a few rows in a batch padded for many, whatever max_q says."""
    c = _case([3], [40], 8, 2, 128, 16, seed=21, pad=200, slopes=True)
    for m in (None, 1, 3, 203, 5000):
        _check(ops, c, max_q=m)
