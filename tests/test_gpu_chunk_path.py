"""The 8-bit projection path as a program runs it: residual norm to e4m3, projection, rotary append, chunk
attention, projection onto the residual, for a prefill of ragged chunks and decode steps behind it; each
stage against 64 bits on the stage's own inputs (the tolerances of the operators' own tests), the steps
from CUDA graphs and other streams against the same calls made eagerly, bit for bit."""

import math

import pytest
import torch

import test_gpu_attn_chunk as attn
import test_gpu_linear as lin
import test_gpu_norm_fp8 as norm
import test_gpu_rope_axes as rope

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
HID, HQ, HKV, D, P, R = 512, 8, 2, 64, 16, 32
AXES = tuple(i % 3 for i in range(R))


@pytest.fixture(scope="module")
def ops():
    from okc_b200 import ops
    return ops


class Layer:
    def __init__(self, B, width, seed):
        g = torch.Generator().manual_seed(seed)
        N = (HQ + 2 * HKV) * D
        rnd = lambda *s: torch.randn(*s, generator=g)
        self.w_norm = (1 + 0.1 * rnd(HID)).to(torch.bfloat16).cuda()
        self.w_qkv = (rnd(N, HID) * 90).clamp(-448, 448).to(E4M3).cuda()
        self.s_qkv = ((0.5 + torch.rand(N, generator=g)) / (90 * HID ** 0.5)).cuda()
        self.w_out = (rnd(HID, HQ * D) / (HQ * D) ** 0.5).to(torch.bfloat16).cuda()
        self.freq = (1.0 / (1e4 ** (torch.arange(R).float() / R))).cuda()
        pool = B * width + 1
        self.table = torch.randperm(pool, generator=g)[:B * width].to(torch.int32).view(B, width).cuda()
        self.k = torch.zeros(pool, P, HKV, D, dtype=torch.uint8).view(E4M3).cuda()
        self.v = self.k.clone()
        self.ks = torch.full((HKV,), 0.02).cuda()
        self.vs = torch.full((HKV,), 0.03).cuda()

    def step(self, ops, x, stream, pos, cu, lens, max_q, stages=None):
        """One layer; the stream is updated in place.  `stages`: a dict that takes what each stage returned."""
        T = x.shape[0]
        h, hs, s = ops.add_rmsnorm_fp8(x, self.w_norm, 1e-6, stream, residual_out=stream)
        qkv = ops.linear(h, self.w_qkv, hs, self.s_qkv)
        q = ops.rope_axes_kv_append(qkv, pos, AXES, self.freq, cu, lens, self.table, self.k, self.v, self.ks, self.vs,
                                    HQ, HKV, D, half=True)
        o = ops.attn_chunk(q, self.k, self.v, self.table, cu, lens, self.ks, self.vs, 1 / math.sqrt(D), softcap=30.0,
                           max_q=max_q)
        if stages is not None:
            stages.update(h=h, hs=hs, s=s.clone(), qkv=qkv, q=q, o=o)
        return ops.linear(o.view(T, HQ * D), self.w_out, residual=stream, out=stream)


def _inputs(new, old, seed):
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32).cuda()
    lens = torch.tensor([n + o for n, o in zip(new, old)], dtype=torch.int32).cuda()
    pos = torch.randint(0, 3000, (3, T), generator=g).cuda()
    return (torch.randn(T, HID, generator=g).to(torch.bfloat16).cuda(), torch.randn(T, HID, generator=g).cuda(), pos, cu, lens)


def test_a_prefill_and_decode_steps(ops):
    layer = Layer(3, 16, seed=1)
    old = [0, 0, 0]
    for i, new in enumerate(([5, 130, 40], [1, 1, 1], [3, 1, 4])):
        x, stream, pos, cu, lens = _inputs(new, old, seed=i)
        old = [a + b for a, b in zip(old, new)]
        stream0, k0, v0 = stream.clone(), layer.k.clone(), layer.v.clone()
        st = {}
        y = layer.step(ops, x, stream, pos, cu, lens, max(new), st)
        assert y is stream
        for tag in ("linear", "rope_axes", "attn_chunk"):
            assert ops.read_device_error(tag) == 0
        c = {k: v.cpu() for k, v in st.items()}
        norm._check((st["h"], st["hs"], st["s"]), x.cpu(), layer.w_norm.cpu(), stream0.cpu(), False)
        lin._check(st["qkv"], {"x": c["h"], "w": layer.w_qkv.cpu(), "x_scale": c["hs"], "w_scale": layer.s_qkv.cpu()}, None)
        cache = {"page_table": layer.table.cpu(), "cu_q": cu.cpu(), "seq_lens": lens.cpu(), "k_scale": layer.ks.cpu(),
                 "v_scale": layer.vs.cpu()}
        rope._run_and_check(ops, {"qkv": c["qkv"], "positions": pos.cpu(), "axes": AXES, "inv_freq": layer.freq.cpu(),
                                  "k_cache": k0.cpu(), "v_cache": v0.cpu(), **cache}, HQ, HKV, D, True)
        attn._close(st["o"], {"q": c["q"], "k_cache": layer.k.cpu(), "v_cache": layer.v.cpu(), "sm_scale": 1 / math.sqrt(D),
                              "softcap": 30.0, **cache})
        lin._check(stream, {"x": c["o"].view(-1, HQ * D), "w": layer.w_out.cpu(), "residual": c["s"]}, None)


def _decoder(ops, seed, B=4):
    """(layer, static inputs, step): every call of `step` decodes one token a request."""
    layer = Layer(B, 8, seed)
    x, stream, pos, cu, lens = _inputs([1] * B, [7 * b + seed for b in range(B)], seed)
    layer.k.view(torch.uint8).random_(0, 120)
    layer.v.view(torch.uint8).random_(0, 120)

    def step():
        layer.step(ops, x, stream, pos, cu, lens, 1)
        lens.add_(1)
        pos.add_(1)
        x.copy_(stream)

    return layer, (x, stream, pos, cu, lens), step


def _state(layer, inputs):
    return [t.clone() for t in (layer.k, layer.v) + inputs]


def _restore(layer, inputs, state):
    for t, s in zip((layer.k, layer.v) + inputs, state):
        t.copy_(s)


def _equal(layer, inputs, state):
    return all(torch.equal(t.view(torch.uint8) if t.dtype == E4M3 else t, s.view(torch.uint8) if s.dtype == E4M3 else s)
               for t, s in zip((layer.k, layer.v) + inputs, state))


def test_graphs_replayed_side_by_side(ops):
    """Two captured decode steps, replayed alternately and then at once on two streams, give what eager calls give."""
    runs = []
    for seed in (3, 4):
        layer, inputs, step = _decoder(ops, seed)
        first = _state(layer, inputs)
        for _ in range(6):
            step()
        want = _state(layer, inputs)
        _restore(layer, inputs, first)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        _restore(layer, inputs, first)
        runs.append((layer, inputs, first, want, graph))
    for _ in range(6):
        for r in runs:
            r[4].replay()
    torch.cuda.synchronize()
    assert all(_equal(r[0], r[1], r[3]) for r in runs)
    for r in runs:
        _restore(*r[:3])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(6):
        for r, s in zip(runs, streams):
            with torch.cuda.stream(s):
                r[4].replay()
    torch.cuda.synchronize()
    assert all(_equal(r[0], r[1], r[3]) for r in runs)
    for tag in ("linear", "rope_axes", "attn_chunk"):
        assert ops.read_device_error(tag) == 0


def test_two_streams_at_once(ops):
    """Eager steps of two batches interleaved on two streams, neither of them the default one."""
    runs = []
    for seed in (5, 6):
        layer, inputs, step = _decoder(ops, seed)
        first = _state(layer, inputs)
        for _ in range(5):
            step()
        want = _state(layer, inputs)
        _restore(layer, inputs, first)
        runs.append((layer, inputs, want, step, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, _, _, step, s in runs:
            with torch.cuda.stream(s):
                step()
    torch.cuda.synchronize()
    assert all(_equal(layer, inputs, want) for layer, inputs, want, _, _ in runs)


def test_a_captured_prefill(ops):
    """Chunks on the tensor-memory kernel, their keys split, from a graph: equal to the eager call each time."""
    for n, old in ((150, 3000), (600, 64)):
        c = attn._cuda(attn._case([n], [old], HQ, HKV, D, P, seed=n, cap=30.0, slopes=True))
        out = torch.empty_like(c["q"])
        want = ops.attn_chunk(**c, max_q=n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attn_chunk(**c, max_q=n, out=out)
        for _ in range(3):
            out.fill_(7.0)
            graph.replay()
            assert torch.equal(out, want)


def test_a_first_call_inside_a_capture_is_refused(ops):
    from okc_b200._lib import OkcError
    c = attn._cuda(attn._case([1], [3], HQ, HKV, D, P))
    ops.attn_chunk(**c, max_q=1)
    kept = ops._WS.pop((0, "attn_chunk"))
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(OkcError, match="capture"):
                ops.attn_chunk(**c, max_q=1)
    finally:
        ops._WS[(0, "attn_chunk")] = kept


@pytest.mark.parametrize("n", [1, 90])
def test_a_cache_past_32_bits(ops, n):
    """Pages whose elements lie beyond 2^32: appended and read through both attention kernels."""
    far = 2 ** 32 // (P * HKV * D) + 5
    free = torch.cuda.mem_get_info()[0]
    if free < 5 * far * P * HKV * D:
        pytest.skip("needs 21 GB of device memory")
    big = [torch.empty(far + 12, P, HKV, D, dtype=E4M3, device="cuda") for _ in range(2)]
    layer = Layer(2, 6, seed=9)
    pages = layer.k.shape[0]
    x, stream, pos, cu, lens = _inputs([n, 1], [3, 60], seed=9)
    for t in (layer.k, layer.v):
        t.view(torch.uint8).random_(0, 120)
    for b, t in zip(big, (layer.k, layer.v)):
        b.view(torch.uint8)[far - 1:far - 1 + pages] = t.view(torch.uint8)
    s0 = stream.clone()
    want = layer.step(ops, x, stream, pos, cu, lens, n).clone()
    small = (layer.k, layer.v)
    layer.k, layer.v, layer.table = big[0], big[1], layer.table + (far - 1)
    got = layer.step(ops, x, s0, pos, cu, lens, n)
    assert torch.equal(got, want)
    for b, t in zip(big, small):
        assert torch.equal(b.view(torch.uint8)[far - 1:far - 1 + pages], t.view(torch.uint8))
    assert ops.read_device_error("attn_chunk") == 0 and ops.read_device_error("rope_axes") == 0


def test_an_output_past_32_bits(ops):
    M, N, K = 70000, 32768, 64
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    w = torch.randn(N, K, device="cuda").to(torch.bfloat16)
    y = ops.linear(x, w)
    rows = [0, 255, 65535, 65536, M - 1]
    lin._check(y[rows], {"x": x[rows].cpu(), "w": w.cpu()}, None)


def test_quotients_and_overflow_of_the_append(ops):
    """The append's e4m3 quotients are those of an fp32 division, overflow is NaN: every bf16 value, scales of
    each kind, against rope_kv_append, which divides."""
    hq, hkv, d, p = 1, 4, 64, 16
    vals = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # wraps: every bit pattern
    T = 65536 // (hkv * d)
    for scales in ([1.0, 0.37, 3.0, 0.0123], [2.0 ** -70, 2.0 ** 70, 2.0 ** -59, 1e-38], [448.0, 1 / 3, 464.0, 1e20]):
        qkv = torch.zeros(T, hq + 2 * hkv, d, dtype=torch.bfloat16)
        qkv[:, hq + hkv:] = vals.view(T, hkv, d)
        qkv = qkv.view(T, -1).cuda()
        lens = torch.arange(1, T + 1, dtype=torch.int32)
        table = torch.arange(T, dtype=torch.int32).view(T, 1).cuda()
        lens = torch.ones(T, dtype=torch.int32).cuda()
        pos = torch.zeros(1, T, dtype=torch.int64).cuda()
        freq = torch.ones(d // 2).cuda()
        ks = torch.ones(hkv).cuda()
        vs = torch.tensor(scales).cuda()
        caches = [torch.zeros(T, p, hkv, d, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(4)]
        ops.rope_axes_kv_append(qkv, pos, (0,) * (d // 2), freq, torch.arange(T + 1, dtype=torch.int32).cuda(), lens, table,
                                caches[0], caches[1], ks, vs, hq, hkv, d)
        ops.rope_kv_append(qkv, pos[0], table, caches[2], caches[3], ks, vs, hq, hkv, d, freq)
        a, b = (t.view(torch.uint8)[:, 0].cpu() for t in (caches[1], caches[3]))
        nan = (a & 0x7F) == 0x7F
        assert torch.equal(nan, (b & 0x7F) == 0x7F)
        assert torch.equal(a[~nan], b[~nan])


def test_odd_arguments_are_refused(ops):
    from okc_b200._lib import OkcError
    c = rope._cuda(rope._case([2], [3], 2, 1, 64, 16, 32, (0,) * 32, seed=1))
    for more in (dict(axes=32), dict(axes=0), dict(axes="a" * 32), dict(axes=(0.0,) * 32), dict(page_table=c["page_table"][0]),
                 dict(page_table=c["page_table"][0, 0])):
        with pytest.raises(OkcError):
            ops.rope_axes_kv_append(**{**c, **more}, Hq=2, Hkv=1, D=64)
    for f, args in ((ops.linear, (torch.zeros(2, 16), torch.zeros(2, 16))), (ops.add_rmsnorm_fp8, (torch.zeros(2, 16), torch.zeros(16), 1e-6))):
        with pytest.raises(OkcError):
            f(*args)  # not on a GPU


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("n", [1, 2, 20, 90])
def test_infinite_and_nan_queries_stay_in_their_rows(ops, n, cap):
    """A row of q with NaN or infinities does not reach its neighbours.  On the short chunks' kernel they do not
    change.  The long chunks' kernel takes the origin of the exponentials and the form of the cap's tanh for
    32 rows together, so that a neighbour's roundings may differ: it is held to the operator's tolerance."""
    cpu = attn._case([n, 2], [70, 9], 8, 2, 64, 16, seed=n, cap=cap)
    c = attn._cuda(cpu)
    o = ops.attn_chunk(**c, max_q=n)
    q = c["q"].clone()
    q[0, 1, 3], q[0, 4, 0], q[n, 5, 7] = float("nan"), float("inf"), float("-inf")
    o2 = ops.attn_chunk(**{**c, "q": q}, max_q=n)
    same = torch.ones(n + 2, 8, dtype=torch.bool, device="cuda")
    same[0, 1] = same[0, 4] = same[n, 5] = False
    if n * 4 <= 64:
        assert torch.equal(o[same], o2[same])
    attn._close(torch.where(same[..., None], o2, o), cpu)
    assert torch.isnan(o2[0, 1].float()).all()


@pytest.mark.parametrize("half", [False, True])
def test_appends_of_thousands_of_tokens(ops, half):
    """Several tokens share a block then: chunk ends inside it, a last block that is not whole, rows behind the last chunk."""
    new, old = [1500, 0, 2, 601], [3, 9, 60, 30]
    c = rope._case(new, old, 7, 1, 64, 16, 16, tuple(i % 3 for i in range(16)), 100000, seed=5, pad=2)
    rope._run_and_check(ops, c, 7, 1, 64, half)
    # one page outside the pool: its tokens are skipped, the others are appended
    from okc_b200 import _lib
    d = rope._cuda(c)
    ops.rope_axes_kv_append(**d, Hq=7, Hkv=1, D=64, half=half)
    e = rope._cuda(c)
    page = int(c["page_table"][0, 40])
    e["page_table"][0, 40] = -1
    ops.rope_axes_kv_append(**e, Hq=7, Hkv=1, D=64, half=half)
    assert ops.read_device_error("rope_axes") == _lib.DEVERR_PAGE
    for t in ("k_cache", "v_cache"):
        want = d[t].view(torch.uint8)
        want[page] = c[t].view(torch.uint8)[page].cuda()
        assert torch.equal(e[t].view(torch.uint8), want)


def test_everything_is_asked_of_the_tensors_device(ops, monkeypatch):
    """With another device current, the size of the scratch, which goes with the device's SMs, and the launches are
    those of the tensors' device.  (The other device is made up: its number is all that is asked of it.)"""
    c = attn._cuda(attn._case([2], [30], HQ, HKV, D, P))
    want = ops.attn_chunk(**c, max_q=2)
    current, seen, real, device = [1], {}, ops._LIB, torch.cuda.device

    class Device(device):
        def __enter__(self):
            current[0] = 0
            return super().__enter__()

        def __exit__(self, *a):
            current[0] = 1
            return super().__exit__(*a)

    class Lib:
        def __getattr__(self, name):
            def f(*args):
                seen[name] = current[0]
                return getattr(real, name)(*args)
            return f

    monkeypatch.setattr(ops, "_LIB", Lib())
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    assert torch.equal(ops.attn_chunk(**c, max_q=2), want)
    assert seen == {"okc_attn_chunk_workspace_bytes": 0, "okc_attn_chunk_fp8": 0}
