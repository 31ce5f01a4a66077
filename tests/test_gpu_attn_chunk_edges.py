"""Chunk attention (ops.attn_chunk) where it is told little or extremes: row tiles without a key, limits and
sentinels of its arguments, caps of every size, weights far below the row's largest.  Tolerances beyond those of
test_gpu_attn_chunk.py stand beside the tests that need them."""

import math

import pytest
import torch

import test_gpu_attn_chunk as attn
from oracle import chunk as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


@pytest.fixture(autouse=True)
def wide_tables():
    """Tables much wider than the requests, so that long chunks go to the long chunks' kernel."""
    attn.WIDE = True
    yield
    attn.WIDE = False


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,Hq,Hkv", [(2600, 8, 8), (700, 2, 1)], ids=["keys-whole", "keys-split"])
def test_row_tiles_without_keys_are_zero(ops, new, Hq, Hkv, D):
    """Whole 256-row tile pairs that see nothing, beside pairs that do, their queries NaN, infinite and large: zeros
    each time, and the other rows as they are without those queries.  2600 rows at 8 heads fill the grid (one
    segment a row), 1400 rows at one head split the keys, of which most rows have few segments."""
    c = attn._case([new], [40], Hq, Hkv, D, 16, seed=D + new)
    rows = 256 * Hkv // Hq  # tokens of a tile pair
    blind = torch.zeros(new, dtype=torch.bool)
    for pair in (0, 2, 3, new // rows):  # the last one is not whole
        blind[pair * rows:(pair + 1) * rows] = True
    c["doc_start"] = torch.where(blind, 10 ** 6, 0).to(torch.int32)
    d = attn._cuda(c)
    blind = blind.cuda()
    d["q"][blind] = 0
    want = ops.attn_chunk(**d, max_q=new)
    assert (want[blind] == 0).all() and torch.isfinite(want.float()).all()
    for value in (float("nan"), float("inf"), 3e38):
        d["q"][blind] = value
        for _ in range(5):
            out = torch.full_like(want, 9.0)
            assert torch.equal(ops.attn_chunk(**d, max_q=new, out=out), want)
    d["seq_lens"][0] = 0  # every row sits before position 0
    for _ in range(5):
        out = torch.full_like(want, 9.0)
        assert (ops.attn_chunk(**d, max_q=new, out=out) == 0).all()
    assert ops.read_device_error("attn_chunk") == 0


@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_query_beside_empty_key_segments(ops, D):
    """A live row of NaN beside rows whose keys lie in the first segment only."""
    c = attn._case([300], [0], 2, 1, D, 16, seed=D)
    d = attn._cuda(c)
    o = ops.attn_chunk(**d, max_q=300)
    d["q"][7, 1] = float("nan")
    for _ in range(5):
        o2 = ops.attn_chunk(**d, max_q=300)
        assert torch.isnan(o2[7, 1].float()).all()
        o2[7, 1] = o[7, 1]
        attn._close(o2, c)


def test_a_long_chunk_behind_a_table_of_a_million_positions(ops):
    """16384 tokens at 64 / 8 heads, the table's width 2^20 positions: what a table cut to the request gives."""
    g = torch.Generator(device="cuda").manual_seed(3)
    T, Hq, Hkv, D, P = 16384, 64, 8, 128, 16
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    c = dict(q=rnd(T, Hq, D).to(torch.bfloat16), k_cache=rnd(T // P, P, Hkv, D).to(attn.E4M3),
             v_cache=rnd(T // P, P, Hkv, D).to(attn.E4M3), cu_q=torch.tensor([0, T], dtype=torch.int32, device="cuda"),
             seq_lens=torch.tensor([T], dtype=torch.int32, device="cuda"), k_scale=torch.ones(Hkv, device="cuda"),
             v_scale=torch.ones(Hkv, device="cuda"), sm_scale=1 / math.sqrt(D), max_q=T)
    table = torch.full((1, 2 ** 20 // P), -1, dtype=torch.int32, device="cuda")
    table[0, :T // P] = torch.randperm(T // P, generator=g, device="cuda").to(torch.int32)
    want = ops.attn_chunk(page_table=table[:, :T // P], **c)
    assert torch.equal(ops.attn_chunk(page_table=table, **c), want)
    assert ops.read_device_error("attn_chunk") == 0 and want.abs().max() > 0


@pytest.mark.parametrize("Hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("n", [1, 3, 40, 300])
def test_the_largest_document_start_is_no_work(ops, Hkv, n):
    """doc_start 2^31 - 1 for rows that see nothing, whole tiles of them and single ones: zeros, in no time."""
    c = attn._case([n, 5], [70, 40], 4 * Hkv, Hkv, 64, 16, seed=n + Hkv)
    for first in (0, 4):  # the second time the first tokens see their keys
        c["doc_start"] = torch.full((n + 5,), 2 ** 31 - 1, dtype=torch.int32)
        c["doc_start"][:first] = 0
        attn._check(ops, c, max_q=n)
        d = attn._cuda(c)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        ops.attn_chunk(**d, max_q=n)
        start.record()
        ops.attn_chunk(**d, max_q=n)
        end.record()
        end.synchronize()
        assert start.elapsed_time(end) < 100  # milliseconds: one empty step for each of 2^31 positions takes seconds


@pytest.mark.parametrize("n", [9, 100])
def test_the_widest_window_with_rows_before_position_0(ops, n):
    """More new tokens than cached ones: the rows before position 0 see nothing, a window of 2^31 - 1 leaves the
    others all their keys."""
    c = attn._case([n, 2], [0, 30], 8, 2, 64, 16, seed=n)
    c["seq_lens"][0] = n - 5
    d = attn._cuda(c)
    want = ops.attn_chunk(**d, max_q=n)
    assert (want[:5] == 0).all() and (want[5:].abs().amax((1, 2)) > 0).all()
    d["window"] = 2 ** 31 - 1
    assert torch.equal(ops.attn_chunk(**d, max_q=n), want)
    assert ops.read_device_error("attn_chunk") == 0


@pytest.mark.parametrize("n", [2, 90])
def test_windows_past_32_bits(ops, n):
    """A window wider than a C int is one that leaves every key, not its low bits; a negative one is refused."""
    from okc_b200._lib import OkcError
    d = attn._cuda(attn._case([n, 1], [40, 30], 8, 2, 64, 16, seed=n))
    want = ops.attn_chunk(**d, max_q=n)
    for window in (2 ** 31, 2 ** 32 + 3, 2 ** 40):
        d["window"] = window
        assert torch.equal(ops.attn_chunk(**d, max_q=n), want)
    d["window"] = 0
    for more in (dict(window=-(2 ** 32)), dict(window=-1), dict(max_q=-(2 ** 32))):
        with pytest.raises(OkcError):
            ops.attn_chunk(**{**d, **more})
    attn._close(ops.attn_chunk(**d, max_q=2 ** 32 + 1), {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()})


@pytest.mark.parametrize("cap", [1e-6, 1e-3, 0.5, 127.0, 129.0, 1000.0, 1030.0, 2e4, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("n,slopes", [(1, False), (5, True), (40, False), (90, True), (300, False)])
def test_caps_of_every_size(ops, n, slopes, cap):
    """A cap far above the scores leaves them as they are.  Scores are under 32: the tanh is within 2^-21 of itself or
    1.2e-7 of the cap where that is at most 1024, so a score is off by 2^-13 at most: inside the tolerance, which
    allows 2^-14 for it beside 2^-11 for the products."""
    c = attn._case([n, 2], [200, 77], 8, 2, 128, 16, seed=n, cap=cap, slopes=slopes)
    attn._check(ops, c, f"cap {cap}", max_q=n)
    c = attn._case([n, 2], [200, 77], 8, 4, 64, 16, seed=n, cap=cap, slopes=slopes)
    attn._check(ops, c, f"cap {cap}", max_q=n)


@pytest.mark.parametrize("cap", [100.0, 130.0, 600.0, 1500.0, 1e5])
@pytest.mark.parametrize("n", [2, 70, 300])
def test_scores_of_hundreds_under_larger_caps(ops, n, cap):
    """Scores of up to 350 on both sides of the polynomials' range; off by 350 * 2^-20 more than in
    test_large_scores, whose 2^-7 allows four times that.  A probability below the f16 normals is off by up to 2^-25 of the
    row's largest: all of the up to 340 keys' together by 340 * 2^-25 of the largest |v|, which shows where the one key
    that a row is about has a value of zero."""
    c = attn._case([2, n], [100, 240], 8, 2, 128, 16, seed=4, cap=cap)
    c["sm_scale"] = 1.0
    o = ops.attn_chunk(**attn._cuda(c), max_q=n).cpu().double()
    want, a = ref.attn_chunk(**c)
    small = 340 * 2.0 ** -25 * float((c["v_cache"].float() * c["v_scale"][:, None]).abs().max())
    assert ((o - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * a + small).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 50.0, 2000.0])
@pytest.mark.parametrize("n,keys", [(1, 4000), (2, 2 ** 20), (5, 333), (300, 4000)])
def test_many_keys_far_below_one(ops, n, keys, cap, D):
    """One key 18 units above all others, its value 0 where theirs is 1: the output is the others' share.  A probability
    is off by 2^-11 of itself or 2^-32 of the row's largest, whichever is more, the output by 2^-9 more."""
    Hq, P = 2, 16
    pages = -(-keys // P)
    for at in (0, keys // 2, keys - n):  # every row sees it
        k = torch.zeros(pages, P, 1, D)
        v = torch.ones(pages, P, 1, D)
        k[at // P, at % P, 0, 1], v[at // P, at % P] = 18.0, 0.0
        q = torch.zeros(n, Hq, D, dtype=torch.bfloat16)
        q[..., 1] = 1.0
        one = torch.ones(1, device="cuda")
        o = ops.attn_chunk(q.cuda(), k.cuda().to(attn.E4M3), v.cuda().to(attn.E4M3),
                           torch.nn.functional.pad(torch.arange(pages, dtype=torch.int32), (0, 4096), value=-1).view(1, -1).cuda(),
                           torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([keys], dtype=torch.int32).cuda(), one, one,
                           1.0, softcap=cap, max_q=n).cpu().double()
        others = (torch.arange(n).double() + keys - n).view(n, 1, 1)  # keys that a row sees, but one
        share = others * math.exp(-(cap * math.tanh(18 / cap) if cap else 18.0))
        want = share / (1 + share)
        assert ((o - want).abs() <= (2.0 ** -9 + 2.0 ** -11 + 2.0 ** -16) * want + others * 2.0 ** -32).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hkv,kind", [(1216, 2, "even"), (1216, 2, "rising"), (1216, 2, "slopes"), (256, 8, "rising"),
                                        (256, 8, "cap")])
def test_sums_over_a_million_keys(ops, T, Hkv, kind, D):
    """Values that are the same at every position: so is the output, whatever the weights.  The tensor core's truncation
    takes at most 2^-22 of a sum for 16 keys (a unit of it and one for the products' alignment), and 131072 keys go into one
    sum: 2^-9, and 2^-9 for the rounding to bf16.  1216 tokens at 2 / 16 heads fill the grid, 256 at 8 / 64 split the
    keys in two.  Scores that rise with the position move the origin of the exponentials behind sums that are set
    aside; some rows see their first key after 600000."""
    n, P, G = 2 ** 20, 16, 8
    g = torch.Generator(device="cuda").manual_seed(D + T)
    k = torch.randn(n // P, P, Hkv, D, generator=g, device="cuda", dtype=torch.float16)
    q = torch.randn(T, G * Hkv, D, generator=g, device="cuda")
    if kind == "rising":
        k[..., 0] = 12 * (torch.arange(n, device="cuda", dtype=torch.float32).view(n // P, P, 1) / n).half()
        q[..., 0] = 24 * (8 if D == 64 else 11) / 8
    col = 2.0 ** (torch.arange(D) % 5 - 2).float() * (1 - 2.0 * (torch.arange(D) % 2)) * (1 + torch.arange(D) % 3 / 4)
    v = col.to(attn.E4M3).cuda().expand(n // P, P, Hkv, D).contiguous()
    one = torch.ones(Hkv, device="cuda")
    first = torch.zeros(T, dtype=torch.int32)
    first[::7] = 600000
    more = {"slopes": dict(slopes=torch.zeros(G * Hkv, device="cuda")), "cap": dict(softcap=5.0)}.get(kind, {})
    for _ in range(2):
        o = ops.attn_chunk(q.to(torch.bfloat16), k.to(attn.E4M3), v, torch.arange(n // P, dtype=torch.int32, device="cuda").view(1, -1),
                           torch.tensor([0, T], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda"),
                           one, one, 1 / math.sqrt(D), doc_start=first.cuda(), max_q=T, **more)
        assert (o.cpu().float() / col - 1).abs().max() <= 2.0 ** -8
    assert ops.read_device_error("attn_chunk") == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["plain", "cap", "slopes"])
def test_long_contexts_beside_short_chunks(ops, D, kind):
    """A chunk behind 300000 positions, whose sums are set aside in scratch that the short chunks of the same call take
    behind it, against 64 bits on rows of each, with random values, a rising origin, pages in any order and a NaN value
    that some rows see; from a graph twice, and on another stream, the same bits.  The operator's tolerance, and 2^-9
    of the sums for the tensor core's truncation."""
    Hq, Hkv, P, n = 32, 4, 16, [1300, 1, 3]
    full = [300000, 6, 250000]
    g = torch.Generator(device="cuda").manual_seed(D)
    width = -(-max(full) // P) + 2
    pool = 3 * width
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    k = rnd(pool, P, Hkv, D).to(attn.E4M3)
    v = rnd(pool, P, Hkv, D).to(attn.E4M3)
    table = torch.randperm(pool, generator=g, device="cuda").to(torch.int32).view(3, width)
    rise = (torch.arange(width * P, device="cuda") * (20.0 / (width * P))).view(width, P, 1)
    for b in range(3):
        k[table[b].long(), :, :, 0] = rise.expand(width, P, Hkv).to(attn.E4M3)
    T = sum(n)
    q = rnd(T, Hq, D)
    q[..., 0] = 1.0 * D ** 0.5
    q = q.to(torch.bfloat16)
    cu = torch.tensor([0, 1300, 1301, 1304], dtype=torch.int32, device="cuda")
    ks, vs = torch.full((Hkv,), 0.75, device="cuda"), torch.full((Hkv,), 1.25, device="cuda")
    more = {"plain": {}, "cap": dict(softcap=40.0), "slopes": dict(slopes=2.0 ** (-14.0 - torch.arange(Hq, device="cuda") / 8))}[kind]
    call = lambda **kw: ops.attn_chunk(q, k, v, table, cu, torch.tensor(full, dtype=torch.int32, device="cuda"), ks, vs, 1 / math.sqrt(D),
                                       max_q=1300, **more, **kw)
    o = call()
    lens = torch.tensor(full, dtype=torch.int32, device="cuda")
    for t, b in ((0, 0), (131, 0), (700, 0), (1299, 0), (1300, 1), (1301, 2), (1303, 2)):
        p = full[b] - n[b] + t - int(cu[b])
        j = torch.arange(p + 1, device="cuda")
        page = table[b].long()[j // P]
        for h in (0, 13, 31):
            kk, vv = (x.view(torch.uint8)[page, j % P, h // 8].view(attn.E4M3).float().double() for x in (k, v))
            s = kk @ q[t, h].double() * (0.75 / math.sqrt(D))
            if kind == "cap":
                s = 40 * torch.tanh(s / 40)
            if kind == "slopes":
                s = s - more["slopes"][h].double() * (p - j)
            w = torch.softmax(s, 0)
            want, a = w @ vv * 1.25, w @ vv.abs() * 1.25
            assert ((o[t, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -9.5 + 2.0 ** -9) * a).all(), (t, h)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(o)
    args = (q, k, v, table, cu, lens, ks, vs, 1 / math.sqrt(D))
    with torch.cuda.graph(graph):
        ops.attn_chunk(*args, max_q=1300, out=out, **more)
    for _ in range(2):
        out.fill_(5.0)
        graph.replay()
        assert torch.equal(out, o)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        o2 = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, o) and torch.equal(out, o)
    # position 100000 of the first request: every row of it, and only its head and column
    v.view(torch.uint8)[int(table[0, 100000 // P]), 100000 % P, 2, 7] = 0x7F
    nan = torch.isnan(call().float())
    want = torch.zeros_like(nan)
    want[:1300, 16:24, 7] = True
    assert torch.equal(nan, want)
    assert ops.read_device_error("attn_chunk") == 0


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,P", [(128, 1, 64, 16), (160, 2, 128, 3), (6, 3, 128, 16), (30, 6, 64, 1), (65, 1, 64, 128)])
@pytest.mark.parametrize("kind", [dict(), dict(cap=1500.0, slopes=True, prefix=True), dict(window=33, docs=True)])
def test_other_groups_of_heads(ops, Hq, Hkv, D, P, kind, wide):
    """More query heads a KV head than a short chunk may have rows; head counts that no block of 2, 4 or 8 divides."""
    attn.WIDE = wide
    c = attn._case([1, 4, 0, 9], [0, 90, 3, 200], Hq, Hkv, D, P, seed=Hq, pad=2, **kind)
    for m in (9, None):
        attn._check(ops, c, max_q=m)
    c = attn._case([1], [300], Hq, Hkv, D, P, seed=Hq, **kind)
    attn._check(ops, c, max_q=1)
