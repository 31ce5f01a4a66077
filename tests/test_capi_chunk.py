"""CPU checks of the entry points of the 8-bit projection path and of ragged batches: what they refuse is
refused before any CUDA call (the addresses here are made up), and no rows are no work."""

import pytest

INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    from okc_b200 import _lib
    return _lib.load()


@pytest.fixture(scope="module")
def code():
    from okc_b200 import _lib
    return _lib


NORM = dict(x=16, ldx=512, residual=16, ldr=512, residual_fp32=1, w=16, residual_out=16, ldo=512, q=16, ldq=512, scale=16,
            T=2, H=512, eps=1e-6, unit_offset=0, stream=None)
LINEAR = dict(x=16, ldx=64, w=16, ldw=64, e4m3=1, x_scale=16, w_scale=16, w_scale_one=0, bias=16, act=0, residual=16, ldr=40,
              residual_fp32=0, y=16, ldy=40, out_fp32=0, M=3, N=40, K=64, error=16, stream=None)
ROPE = dict(qkv=16, ldqkv=512, positions=16, ld_pos=2, axes=1, axis_of_pair=bytes(32), inv_freq=16, pairs=32, half=0, cu_q=16,
            seq_lens=16, B=2, page_table=16, table_ld=4, max_pages=4, k_scale=16, v_scale=16, q_out=16, ldq=256, k_cache=16,
            v_cache=16, T=2, Hq=4, Hkv=2, D=64, page_size=16, num_pages=9, error=16, stream=None)
ATTN = dict(q=16, ldq=256, k_cache=16, v_cache=16, page_table=16, table_ld=4, max_pages=4, cu_q=16, seq_lens=16, k_scale=16,
            v_scale=16, slopes=None, prefix_lens=None, doc_start=None, out=16, ldo=256, T=2, B=2, Hq=4, Hkv=2, D=64, page_size=16,
            num_pages=9, sm_scale=0.1, softcap=0.0, window=0, max_q=1, workspace=None, workspace_bytes=0, error=16, stream=None)


def _call(fn, base, **more):
    return fn(*{**base, **more}.values())


def test_norm_refusals(lib, code):
    fn = lib.okc_add_rmsnorm_fp8
    assert _call(fn, NORM, T=0) == code.OKC_OK
    for bad in (dict(x=None), dict(w=None), dict(q=None), dict(scale=None), dict(residual_out=None), dict(T=-1), dict(H=0),
                dict(H=520), dict(H=16400, ldx=16400, ldr=16400, ldo=16400, ldq=16400), dict(ldx=511), dict(ldq=256),
                dict(ldr=16), dict(ldo=16)):
        assert _call(fn, NORM, **bad) in (code.OKC_ERR_INVALID, code.OKC_ERR_ALIGNMENT), bad
    for bad in (dict(x=8), dict(ldx=516), dict(residual=4), dict(w=2), dict(q=4)):
        assert _call(fn, NORM, **bad) == code.OKC_ERR_ALIGNMENT, bad


def test_linear_refusals(lib, code):
    fn = lib.okc_linear
    assert _call(fn, LINEAR, M=0) == code.OKC_OK
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(error=None), dict(M=-1), dict(N=0), dict(K=0), dict(K=72, ldx=80, ldw=80),
                dict(act=5), dict(act=-1), dict(ldx=48), dict(ldw=32), dict(ldy=39), dict(ldr=1)):
        assert _call(fn, LINEAR, **bad) == code.OKC_ERR_INVALID, bad
    for bad in (dict(x=8), dict(w=4), dict(ldx=72), dict(ldw=72), dict(y=1), dict(residual=1), dict(residual=2, residual_fp32=1),
                dict(y=2, out_fp32=1)):
        assert _call(fn, LINEAR, **bad) == code.OKC_ERR_ALIGNMENT, bad


def test_rope_refusals(lib, code):
    fn = lib.okc_rope_axes_kv_append
    assert _call(fn, ROPE, T=0) == code.OKC_OK
    for name in ("qkv", "positions", "axis_of_pair", "inv_freq", "cu_q", "seq_lens", "page_table", "k_scale", "v_scale", "q_out",
                 "k_cache", "v_cache", "error"):
        assert _call(fn, ROPE, **{name: None}) == code.OKC_ERR_INVALID, name
    for bad in (dict(T=-1), dict(B=0), dict(Hq=0), dict(Hkv=0), dict(D=60), dict(D=264), dict(pairs=0), dict(pairs=12), dict(pairs=40),
                dict(axes=0), dict(axes=5), dict(page_size=0), dict(num_pages=0), dict(max_pages=0), dict(table_ld=3), dict(ld_pos=1),
                dict(ldqkv=504), dict(ldq=248), dict(axis_of_pair=bytes(31) + b"\x01")):
        assert _call(fn, ROPE, **bad) == code.OKC_ERR_INVALID, bad
    for bad in (dict(qkv=8), dict(q_out=8), dict(ldqkv=516), dict(ldq=260), dict(k_cache=4), dict(v_cache=4), dict(positions=4)):
        assert _call(fn, ROPE, **bad) == code.OKC_ERR_ALIGNMENT, bad


def test_attention_refusals(lib, code):
    fn = lib.okc_attn_chunk_fp8
    assert _call(fn, ATTN, T=0) == code.OKC_OK
    for name in ("q", "k_cache", "v_cache", "page_table", "cu_q", "seq_lens", "k_scale", "v_scale", "out", "error"):
        assert _call(fn, ATTN, **{name: None}) == code.OKC_ERR_INVALID, name
    for bad in (dict(T=-1), dict(B=0), dict(B=2049), dict(Hq=0), dict(Hkv=0), dict(Hq=3), dict(D=96), dict(page_size=0), dict(num_pages=0),
                dict(max_pages=0), dict(window=-1), dict(max_q=-1), dict(sm_scale=INF), dict(softcap=INF), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(table_ld=3), dict(ldq=248), dict(ldo=248)):
        assert _call(fn, ATTN, **bad) == code.OKC_ERR_INVALID, bad
    for bad in (dict(q=8), dict(out=8), dict(k_cache=8), dict(v_cache=8), dict(ldq=260), dict(ldo=260)):
        assert _call(fn, ATTN, **bad) == code.OKC_ERR_ALIGNMENT, bad
    # rows of the cache, of the work list and of the output are counted in 32 bits
    for bad in (dict(num_pages=2 ** 27), dict(num_pages=2 ** 40), dict(page_size=2 ** 30, num_pages=4),
                dict(T=2 ** 30, Hq=4), dict(T=2 ** 23, Hq=4), dict(T=2 ** 24, max_pages=2 ** 20, table_ld=2 ** 20)):
        assert _call(fn, ATTN, **bad) == code.OKC_ERR_TOO_LARGE, bad
    assert _call(fn, ATTN) == code.OKC_ERR_WORKSPACE
    assert _call(fn, ATTN, workspace=256, workspace_bytes=100) == code.OKC_ERR_WORKSPACE
    assert _call(fn, ATTN, num_pages=2 ** 27 - 1) == code.OKC_ERR_WORKSPACE  # the largest cache


def test_workspace_sizes(lib):
    size = lib.okc_attn_chunk_workspace_bytes
    for bad in ((0, 1, 4, 2, 64), (1, 0, 4, 2, 64), (1, 1, 0, 2, 64), (1, 1, 4, 0, 64), (1, 1, 4, 3, 64), (1, 1, 4, 2, 96)):
        assert size(*bad) == 0
    assert 0 < size(1, 1, 4, 2, 64) <= size(100, 1, 4, 2, 64) and size(100, 9, 4, 2, 64) > 0


def test_wide_tables_are_taken(lib, code):
    """Tables far wider than the requests: what limits them is the work that the kernels number, not the width alone.
    (Past all the other checks these calls stop at the missing workspace.)"""
    fn = lib.okc_attn_chunk_fp8
    big = dict(Hq=64, Hkv=8, D=128, ldq=8192, ldo=8192)
    for good in (dict(T=16384, B=1, max_q=16384, max_pages=2 ** 16),  # one long chunk, a table of 2^20 positions
                 dict(T=16384, B=1, max_q=0, max_pages=2 ** 26),
                 dict(T=16384, B=64, max_q=8192, max_pages=2 ** 16),
                 dict(T=2048 * 8, B=2048, max_q=8, max_pages=2 ** 16),  # verify blocks: one tile each
                 dict(T=2048 * 8, B=2048, max_q=8, max_pages=2 ** 18),
                 dict(T=2048, B=2048, max_q=1, max_pages=2 ** 18)):
        assert _call(fn, ATTN, **big, **good, table_ld=good["max_pages"]) == code.OKC_ERR_WORKSPACE, good
    for bad in (dict(T=2048 * 8, B=2048, max_q=8, max_pages=2 ** 21), dict(T=2048, B=2048, max_q=0, max_pages=2 ** 26)):
        assert _call(fn, ATTN, **big, **bad, table_ld=bad["max_pages"]) == code.OKC_ERR_TOO_LARGE, bad


def test_caps_out_of_range_are_refused(lib, code):
    fn = lib.okc_attn_chunk_fp8
    for cap in (1e-7, 1e-30, 1.1e12, 3e38):
        assert _call(fn, ATTN, softcap=cap) == code.OKC_ERR_INVALID, cap
    for cap in (0.0, 1.01e-6, 30.0, 9.9e11):
        assert _call(fn, ATTN, softcap=cap) == code.OKC_ERR_WORKSPACE, cap
