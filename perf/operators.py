"""Cases of the quantised projection path and of the ragged attention path, with plain torch forms.

Four operators that a layer with an e4m3 cache calls one after the other:

  norm    ops.add_rmsnorm_fp8       residual add + RMSNorm, the output in e4m3 with one scale per row
  linear  ops.linear                act(x w^T * x_scale * w_scale + bias) + residual, e4m3 or bf16 operands
  rope    ops.rope_axes_kv_append   rotary positions with several axes, keys and values appended to the paged cache
  attn    ops.attn_chunk            ragged chunks of new tokens over the paged cache: tanh cap, distance bias, prefix
                                    and document masks, sliding window

`listed()` gives the cases that stand for real use, `draw(rng)` more of the same ranges.  `run` computes a case in
elementary torch operations, or with `own` set through the package's operators; `exact` in 64 bits from the
definitions.
"""

import math
import random

import numpy as np
import torch

own = False

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decode step, the stream in bf16: latency
        {"name": "norm_t1_h8192", "op": "norm", "T": 1, "H": 8192, "stream": "bf16", "unit": False},
        # a prefill block with the fp32 stream of a gated-residual layer: bandwidth
        {"name": "norm_t8192_h8192_f32", "op": "norm", "T": 8192, "H": 8192, "stream": "f32", "unit": True},
        # the QKV projection of one token: a pure weight stream
        {"name": "linear_m1_e4m3", "op": "linear", "M": 1, "N": 10240, "K": 8192, "dtype": "e4m3", "act": "none",
         "bias": True, "residual": "none", "out": "bf16"},
        # the O projection of a decode batch, added to the stream
        {"name": "linear_m128_e4m3_res", "op": "linear", "M": 128, "N": 8192, "K": 8192, "dtype": "e4m3",
         "act": "none", "bias": False, "residual": "bf16", "out": "bf16"},
        # a prefill block through a wide e4m3 projection: tensor-core bound
        {"name": "linear_m8192_e4m3_gelu", "op": "linear", "M": 8192, "N": 10240, "K": 8192, "dtype": "e4m3",
         "act": "gelu_tanh", "bias": True, "residual": "none", "out": "bf16"},
        # odd sizes in bf16, a ragged token count and an output width that is no multiple of a tile
        {"name": "linear_m777_bf16_odd", "op": "linear", "M": 777, "N": 4099, "K": 4104, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": "f32", "out": "f32"},
        # a decode batch, three axes in sections, rotating interleaved pairs
        {"name": "rope_b128_d128", "op": "rope", "B": 128, "n": 1, "ctx": 500, "Hq": 64, "Hkv": 8, "D": 128, "P": 16,
         "rot": 128, "order": "sections", "half": False, "far": 0, "lens": 1},
        # images and video in a prefill block, axes in turn, half-split pairs, part of the head turned
        {"name": "rope_t8000_d128_far", "op": "rope", "B": 5, "n": 1600, "ctx": 700, "Hq": 28, "Hkv": 4, "D": 128,
         "P": 16, "rot": 96, "order": "turns", "half": True, "far": 1000000, "lens": 2},
        # one request decoding far into a long context, capped scores and a distance bias, page 1
        {"name": "attn_b1_ctx80k_d64", "op": "attn", "B": 1, "n": 1, "ctx": 81919, "Hq": 16, "Hkv": 2, "D": 64, "P": 1,
         "cap": 30.0, "slopes": True, "window": 0, "prefix": False, "docs": False, "lens": 3},
        # a decode batch with ragged contexts and capped scores: the cache's bandwidth
        {"name": "attn_b128_decode_cap", "op": "attn", "B": 128, "n": 1, "ctx": 8192, "Hq": 64, "Hkv": 8, "D": 128,
         "P": 16, "cap": 50.0, "slopes": False, "window": 0, "prefix": False, "docs": False, "lens": 4},
        # new tokens of ragged lengths over a cached context, some after a prefix that all see, packed documents
        {"name": "attn_b6_mixed_docs", "op": "attn", "B": 6, "n": 901, "ctx": 2500, "Hq": 28, "Hkv": 4, "D": 128,
         "P": 16, "cap": 0.0, "slopes": True, "window": 0, "prefix": True, "docs": True, "lens": 5},
        # a long prefill chunk behind a cached context, capped scores: tensor-core bound
        {"name": "attn_b1_chunk4096_cap", "op": "attn", "B": 1, "n": 4096, "ctx": 4096, "Hq": 64, "Hkv": 8, "D": 128,
         "P": 16, "cap": 50.0, "slopes": False, "window": 0, "prefix": False, "docs": False, "lens": 6},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "rope", "attn", "attn"))
    if op == "norm":
        H = 16 * _log(rng, 4, 1024)
        return {"op": op, "T": _log(rng, 1, min(16384, 8192 * 8192 // H)), "H": H, "stream": rng.choice(("none", "bf16", "f32")),
                "unit": rng.random() < 0.5}
    if op == "linear":
        dtype = rng.choice(("e4m3", "e4m3", "bf16"))
        K = (16 if dtype == "e4m3" else 8) * _log(rng, 8, 1024)
        N = _log(rng, 64, 28672)
        M = _log(rng, 1, max(1, min(8192, 8192 * 10240 * 8192 // (2 * N * K))))
        return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype, "act": rng.choice(ACTS), "bias": rng.random() < 0.5,
                "residual": rng.choice(("none", "bf16", "f32")), "out": rng.choice(("bf16", "f32"))}
    D = rng.choice((64, 128))
    Hkv = rng.choice((1, 2, 4, 8))
    Hq = Hkv * rng.choice((1, 2, 4, 7, 8, 16) if Hkv < 8 else (1, 2, 4, 7, 8))
    P = rng.choice((1, 16, 16, 64))
    if op == "rope":
        n = _log(rng, 1, 2048)
        return {"op": op, "B": _log(rng, 1, max(1, min(256, 8000 // n))), "n": n, "ctx": _log(rng, 1, 1000), "Hq": Hq, "Hkv": Hkv,
                "D": D, "P": P, "rot": rng.choice((D, D, D // 2)), "order": rng.choice(("sections", "turns")), "half": rng.random() < 0.5,
                "far": rng.choice((0, 50000, 1000000)), "lens": rng.randrange(1 << 20)}
    n = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
    ctx = _log(rng, 1, 65536 if n == 1 else 6000)
    most = 1 << 31  # scores: below the long chunk's
    rows = max(1, min(most // (Hq * n * (ctx + n)), (1 << 30) // ((ctx + n) * Hkv * D)))
    return {"op": op, "B": min(_log(rng, 1, 256), rows), "n": n, "ctx": ctx, "Hq": Hq, "Hkv": Hkv, "D": D, "P": P,
            "cap": rng.choice((0.0, 20.0, 50.0)), "slopes": rng.random() < 0.4, "window": rng.choice((0, 0, 128, 1000, 2048)),
            "prefix": n > 1 and rng.random() < 0.4, "docs": n > 1 and rng.random() < 0.4, "lens": rng.randrange(1 << 20)}


def lengths(case):
    """Per request: (new tokens, tokens in the cache with them).  The first request has the full sizes."""
    rng = random.Random(case["lens"])
    B, n, ctx = case["B"], case["n"], case["ctx"]
    new = [n] + [rng.randint(max(1, n // 8), n) for _ in range(B - 1)]
    old = [ctx] + [rng.randint(ctx // 8, ctx) for _ in range(B - 1)]
    return new, [a + b for a, b in zip(new, old)]


def masks(case):
    """Per request: the prefix that every token sees; per token: the first position of its document (or 0)."""
    rng = random.Random(case["lens"] + 1)
    new, full = lengths(case)
    prefix = [rng.randint(0, f) if case["prefix"] else 0 for f in full]
    first = []
    for n, f in zip(new, full):
        at, start = f - n, 0
        while at < f:  # documents end and begin inside the chunk
            size = rng.randint(1, max(1, n // 2)) if case["docs"] else f
            end = min(f, at + size)
            first += [start] * (end - at)
            at = start = end
    return prefix, first


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _paged(case, g):
    """A shuffled page table, e4m3 caches with per-head scales, and the ragged batch's plan."""
    new, full = lengths(case)
    P, B = case["P"], case["B"]
    pages = [-(-f // P) for f in full]
    pool = sum(pages) + 3
    perm = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((B, max(pages)), dtype=torch.int32, device="cuda")
    starts = np.concatenate([[0], np.cumsum(pages)])
    col = torch.arange(max(pages), device="cuda")
    have = col[None] < torch.tensor(pages, device="cuda")[:, None]
    table[have] = perm[(torch.tensor(starts[:-1].copy(), device="cuda")[:, None] + col[None])[have]]
    shape = (pool, P, case["Hkv"], case["D"])
    s = {"table": table, "k_scale": 0.01 + 0.02 * _rand(g, case["Hkv"]), "v_scale": 0.01 + 0.02 * _rand(g, case["Hkv"])}
    for name in ("k", "v"):
        # stored values of unit spread times 1 / scale, well inside the e4m3 range
        s[name + "_cache"] = (_randn(g, *shape, dtype=torch.float16) / s[name + "_scale"].half()[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(
            torch.float8_e4m3fn)
    s["cu_q"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    s["seq_lens"] = torch.tensor(full, dtype=torch.int32, device="cuda")
    return s


def _axes(case):
    """The axis (time, height, width) that turns each pair."""
    R = case["rot"] // 2
    if case["order"] == "sections":
        a = R // 4
        return tuple([0] * a + [1] * ((R - a) // 2) + [2] * (R - a - (R - a) // 2))
    return tuple(i % 3 for i in range(R))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "norm":
        s = {"x": _randn(g, case["T"], case["H"]).to(torch.bfloat16),
             "w": (_randn(g, case["H"]) * 0.1 + (0.0 if case["unit"] else 1.0)).to(torch.bfloat16), "res": None}
        if case["stream"] != "none":
            s["res"] = (_randn(g, case["T"], case["H"]) * 4).to(torch.bfloat16 if case["stream"] == "bf16" else torch.float32)
    elif op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s = {"x_scale": None, "w_scale": None, "bias": None, "res": None}
        if case["dtype"] == "e4m3":
            # what a dynamic row scale and a channel scale leave: values up to 448
            s["x"] = (_randn(g, M, K) * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            s["w"] = (_randn(g, N, K) * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            s["x_scale"] = (0.5 + _rand(g, M)) / 100
            s["w_scale"] = (0.5 + _rand(g, N)) / (100 * math.sqrt(K))
        else:
            s["x"] = _randn(g, M, K).to(torch.bfloat16)
            s["w"] = (_randn(g, N, K) / math.sqrt(K)).to(torch.bfloat16)
        if case["bias"]:
            s["bias"] = _randn(g, N).to(torch.bfloat16)
        if case["residual"] != "none":
            s["res"] = _randn(g, M, N).to(torch.bfloat16 if case["residual"] == "bf16" else torch.float32)
    elif op == "rope":
        s = _paged(case, g)
        T = sum(lengths(case)[0])
        s["qkv"] = _randn(g, T, (case["Hq"] + 2 * case["Hkv"]) * case["D"]).to(torch.bfloat16)
        # text runs along all three axes together, an image's rows and columns apart from its time
        base = torch.arange(T, device="cuda") + case["far"] + seed % 97
        patch = torch.randint(0, 64, (3, T), generator=g, device="cuda")
        image = _rand(g, T) < 0.5
        s["positions"] = torch.where(image[None], base[None] + patch, base[None]).contiguous()
        R = case["rot"] // 2
        s["inv_freq"] = 1.0 / (5e5 ** (torch.arange(R, device="cuda").float() / R))
        s["axes"] = _axes(case)
        s["axis_of"] = torch.tensor(s["axes"], device="cuda")
    else:
        s = _paged(case, g)
        T = sum(lengths(case)[0])
        s["q"] = (_randn(g, T, case["Hq"], case["D"]) * 2).to(torch.bfloat16)
        prefix, first = masks(case)
        s["prefix"] = torch.tensor(prefix, dtype=torch.int32, device="cuda") if case["prefix"] else None
        s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda") if case["docs"] else None
        s["slopes"] = None
        if case["slopes"]:  # a geometric series over the heads, as distance biases have it
            s["slopes"] = 2.0 ** (-8.0 * (torch.arange(case["Hq"], device="cuda") + 1).float() / case["Hq"])
        s["most"] = case["n"]
    return {"case": case, **s}


# ------------------------------------------------------------------------- plain forms
def _act(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * (1 / math.sqrt(2))))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _norm(s):
    c = s["case"]
    h, stream = s["x"].float(), None
    if s["res"] is not None:
        stream = (h + s["res"].float()).to(s["res"].dtype)
        h = stream.float()
    g = s["w"].float() + (1.0 if c["unit"] else 0.0)
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * g
    top = y.abs().amax(1)
    scale = torch.where(top == 0, torch.ones_like(top), top / E4M3_MAX)
    q = (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, scale, stream


def _linear(s):
    c = s["case"]
    y = s["x"].float() @ s["w"].float().t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None] * s["w_scale"][None]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _act(y, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(torch.bfloat16 if c["out"] == "bf16" else torch.float32)


def _token_places(s, T):
    """Per token: its request, and its position in the request's cache."""
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["cu_q"][1:].long(), t, right=True)
    return b, s["seq_lens"][b].long() - s["cu_q"][b + 1].long() + t


def _rope(s):
    c = s["case"]
    Hq, Hkv, D, P, R = c["Hq"], c["Hkv"], c["D"], c["P"], c["rot"] // 2
    T = s["qkv"].shape[0]
    x = s["qkv"].float().view(T, Hq + 2 * Hkv, D)
    angle = s["positions"][s["axis_of"]].double().t() * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    qk = x[:, :Hq + Hkv]
    if c["half"]:
        a, b = qk[..., :R], qk[..., R:2 * R]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos, qk[..., 2 * R:]], -1)
    else:
        a, b = qk[..., 0:2 * R:2], qk[..., 1:2 * R:2]
        turned = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), qk[..., 2 * R:]], -1)
    b, pos = _token_places(s, T)
    page, at = s["table"][b, pos // P].long(), pos % P
    s["k_cache"].view(torch.uint8)[page, at] = (turned[:, Hq:] / s["k_scale"][:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    s["v_cache"].view(torch.uint8)[page, at] = (x[:, Hq + Hkv:] / s["v_scale"][:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return turned[:, :Hq].to(torch.bfloat16), s["k_cache"], s["v_cache"]


def _attn(s):
    c = s["case"]
    Hq, Hkv, D, P, n, B = c["Hq"], c["Hkv"], c["D"], c["P"], c["n"], c["B"]
    T, L = s["q"].shape[0], s["table"].shape[1] * P
    b, pos = _token_places(s, T)
    i = torch.arange(T, device="cuda") - s["cu_q"][b].long()
    # requests side by side, padded to the longest
    q = torch.zeros((B, n, Hkv, Hq // Hkv, D), device="cuda")
    q[b, i] = s["q"].float().view(T, Hkv, Hq // Hkv, D)
    j = torch.arange(L, device="cuda")
    slot = (s["table"].long()[:, :, None] * P + torch.arange(P, device="cuda")).view(B, L)
    k = s["k_cache"].view(torch.uint8).view(-1, Hkv, D)[slot].view(torch.float8_e4m3fn).float() * s["k_scale"][:, None]
    p = torch.full((B, n), -1, device="cuda", dtype=torch.long)
    p[b, i] = pos
    hi = p + 1
    if s["prefix"] is not None:
        hi = torch.maximum(hi, s["prefix"].long()[:, None])
    hi = torch.minimum(hi, s["seq_lens"].long()[:, None])
    lo = torch.zeros_like(p)
    if c["window"]:
        lo = torch.clamp(p + 1 - c["window"], min=0)
    if s["first"] is not None:
        first = torch.zeros_like(p)
        first[b, i] = s["first"].long()
        lo = torch.maximum(lo, first)
    seen = (j >= lo[..., None]) & (j < hi[..., None])
    w = torch.einsum("bnhgd,blhd->bhgnl", q, k)
    del q, k
    w *= 1 / math.sqrt(D)
    if c["cap"]:
        w.div_(c["cap"]).tanh_().mul_(c["cap"])
    if s["slopes"] is not None:
        w -= s["slopes"].view(Hkv, -1, 1, 1) * (p[..., None] - j).abs().float()[:, None, None]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = w.sum(-1, keepdim=True)
    v = s["v_cache"].view(torch.uint8).view(-1, Hkv, D)[slot].view(torch.float8_e4m3fn).float() * s["v_scale"][:, None]
    v.masked_fill_((j >= s["seq_lens"].long()[:, None])[..., None, None], 0)
    o = torch.einsum("bhgnl,blhd->bhgnd", w, v) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[b, i].to(torch.bfloat16)


def _own(s):
    from okc_b200 import ops

    c = s["case"]
    if c["op"] == "norm":
        return ops.add_rmsnorm_fp8(s["x"], s["w"], 1e-6, residual=s["res"], unit_offset=c["unit"])
    if c["op"] == "linear":
        return ops.linear(s["x"], s["w"], x_scale=s["x_scale"], w_scale=s["w_scale"], bias=s["bias"], act=c["act"], residual=s["res"],
                          out_dtype=torch.bfloat16 if c["out"] == "bf16" else torch.float32)
    if c["op"] == "rope":
        q = ops.rope_axes_kv_append(s["qkv"], s["positions"], s["axes"], s["inv_freq"], s["cu_q"], s["seq_lens"], s["table"], s["k_cache"],
                                    s["v_cache"], s["k_scale"], s["v_scale"], c["Hq"], c["Hkv"], c["D"], half=c["half"])
        return q, s["k_cache"], s["v_cache"]
    return ops.attn_chunk(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu_q"], s["seq_lens"], s["k_scale"], s["v_scale"],
                          1 / math.sqrt(c["D"]), softcap=c["cap"], slopes=s["slopes"], window=c["window"], prefix_lens=s["prefix"],
                          doc_start=s["first"], max_q=s["most"])


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "linear": _linear, "rope": _rope, "attn": _attn}[state["case"]["op"]](state)


# --------------------------------------------------------------------------- the work
def work(case):
    op = case["op"]
    if op == "norm":
        each = {"none": 0, "bf16": 4, "f32": 8}[case["stream"]]  # the stream in and out
        return {"bytes": case["T"] * (case["H"] * (2 + each + 1) + 4) + 2 * case["H"], "flops": 8 * case["T"] * case["H"]}
    if op == "linear":
        M, N, K, size = case["M"], case["N"], case["K"], 1 if case["dtype"] == "e4m3" else 2
        per = {"none": 0, "bf16": 2, "f32": 4}[case["residual"]] + (2 if case["out"] == "bf16" else 4)
        return {"bytes": size * K * (M + N) + M * N * per + (4 * (M + N) if size == 1 else 0) + (2 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    new, full = lengths(case)
    T, D, Hq, Hkv = sum(new), case["D"], case["Hq"], case["Hkv"]
    if op == "rope":
        return {"bytes": T * D * (2 * (Hq + 2 * Hkv) + 2 * Hq + 2 * Hkv) + T * 24, "flops": 6 * T * (Hq + Hkv) * case["rot"] // 2}
    prefix, first = masks(case)
    pairs = keys = at = 0
    for n, f, pre in zip(new, full, prefix):
        p = np.arange(f - n, f)
        hi = np.minimum(np.maximum(p + 1, pre), f)
        lo = np.array(first[at:at + n])
        if case["window"]:
            lo = np.maximum(lo, p + 1 - case["window"])
        at += n
        pairs += int(np.maximum(hi - lo, 0).sum())
        keys += int(max(0, hi.max() - lo.min()))
    return {"bytes": 4 * T * Hq * D + 2 * keys * Hkv * D + 4 * (T + keys // case["P"]), "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h, stream = s["x"].double(), None
        if s["res"] is not None:
            # the sum in 64 bits; the norm is defined on the stream as it is stored
            stream = h + s["res"].double()
            h = stream.to(s["res"].dtype).double()
        rms = (h.square().sum(1) / case["H"] + 1e-6).sqrt()
        y = h / rms[:, None] * (s["w"].double() + float(case["unit"]))
        top = y.abs().max(1).values
        scale = top.div(448).masked_fill(top == 0, 1.0)
        return y / scale[:, None], scale, stream
    if op == "linear":
        y = torch.mm(s["x"].double(), s["w"].double().T)
        if s["x_scale"] is not None:
            y = torch.outer(s["x_scale"].double(), s["w_scale"].double()) * y
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["act"] == "relu":
            y = y * (y > 0)
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif case["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y if s["res"] is None else y + s["res"].double()
    new, full = lengths(case)
    Hq, Hkv, D, P = case["Hq"], case["Hkv"], case["D"], case["P"]
    if op == "rope":
        x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
        R = case["rot"] // 2
        out = x.clone()
        for i, axis in enumerate(s["axes"]):
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"][axis].double() * s["inv_freq"][i].double())
            u, v = (i, i + R) if case["half"] else (2 * i, 2 * i + 1)
            z = torch.complex(x[:, :Hq + Hkv, u], x[:, :Hq + Hkv, v]) * turn[:, None]
            out[:, :Hq + Hkv, u], out[:, :Hq + Hkv, v] = z.real, z.imag
        k, v = s["k_cache"].float().double(), s["v_cache"].float().double()
        t = 0
        for b in range(case["B"]):
            place = torch.arange(full[b] - new[b], full[b], device="cuda")
            page = s["table"][b].long()[place // P]
            rows = slice(t, t + new[b])
            k[page, place % P] = out[rows, Hq:Hq + Hkv] / s["k_scale"].double()[:, None]
            v[page, place % P] = out[rows, Hq + Hkv:] / s["v_scale"].double()[:, None]
            t += new[b]
        return out[:, :Hq], k, v
    prefix, first = masks(case)
    out = torch.zeros((sum(new), Hq, D), dtype=torch.float64, device="cuda")
    t, G = 0, Hq // Hkv
    for b in range(case["B"]):
        place = torch.arange(full[b], device="cuda")
        page = s["table"][b].long()[place // P]
        k = s["k_cache"][page, place % P].float().double()
        v = s["v_cache"][page, place % P].float().double()
        me = torch.arange(full[b] - new[b], full[b], device="cuda")
        far = place[None] - me[:, None]
        see = (far <= 0) | (place[None] < prefix[b])
        if case["window"]:
            see &= far > -case["window"]
        see &= place[None] >= torch.tensor(first[t:t + new[b]], device="cuda")[:, None]
        for h in range(Hq):
            z = s["q"][t:t + new[b], h].double() @ k[:, h // G].T * (s["k_scale"][h // G].double() / math.sqrt(D))
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                z = z - s["slopes"][h].double() * far.abs()
            z = torch.where(see, z, -math.inf)
            e = torch.exp(z - z.max(1, keepdim=True).values.clamp(min=-1e300)) * see
            out[t:t + new[b], h] = e @ v[:, h // G] * s["v_scale"][h // G].double() / e.sum(1, keepdim=True).clamp(min=1e-300)
        t += new[b]
    return out
