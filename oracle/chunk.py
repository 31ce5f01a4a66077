"""64-bit CPU restatements of the 8-bit projection path and of ragged-batch attention, for the
tests: residual RMSNorm to e4m3, projection with an epilogue, multi-axis rotary append and
masked chunk attention.  Each returns unrounded float64 values (and, where a rounding error is
bounded by them, the sums of magnitudes that the bound needs); none has a counterpart in the
reference, which projects in bf16, rotates with one axis and masks causally."""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def add_rmsnorm(x, w, eps, residual=None, unit_offset=False):
    """(y, scale, s): y unrounded, s rounded to the residual's type (the norm is defined on it)."""
    s = x.double()
    stream = None
    if residual is not None:
        stream = (x.float() + residual.float()).to(residual.dtype)
        s = stream.double()
    g = w.double() + (1.0 if unit_offset else 0.0)
    y = s / (s.square().mean(1, keepdim=True) + eps).sqrt() * g
    top = y.abs().amax(1)
    return y, torch.where(top == 0, torch.ones_like(top), top / E4M3_MAX), stream


def act64(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def linear(x, w, x_scale=None, w_scale=None, bias=None, act=None, residual=None):
    """(y, a): y unrounded, a the sum of |x||w| times the scales (the bound of the accumulation)."""
    x, w = x.float().double(), w.float().double()
    y, a = x @ w.t(), x.abs() @ w.abs().t()
    if x_scale is not None:
        y, a = y * x_scale.double()[:, None], a * x_scale.double().abs()[:, None]
    if w_scale is not None:
        y, a = y * w_scale.double(), a * w_scale.double().abs()
    if bias is not None:
        y = y + bias.double()
    y = act64(y, act)
    return (y if residual is None else y + residual.double()), a


def places(cu_q, seq_lens):
    """Per row: (request, cache position)."""
    out = []
    for b in range(len(seq_lens)):
        n = int(cu_q[b + 1]) - int(cu_q[b])
        out += [(b, int(seq_lens[b]) - n + i) for i in range(n)]
    return out


def rope_axes(qkv, positions, axes, inv_freq, Hq, Hkv, D, half):
    """Turned q and k heads and the v heads, [T, Hq + 2 Hkv, D] float64."""
    T, R = qkv.shape[0], len(axes)
    x = qkv.double().view(T, Hq + 2 * Hkv, D)
    out = x.clone()
    for i, ax in enumerate(axes):
        ang = positions[ax].double() * inv_freq[i].double()
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        u, v = (i, i + R) if half else (2 * i, 2 * i + 1)
        a, b = x[:, :Hq + Hkv, u], x[:, :Hq + Hkv, v]
        out[:, :Hq + Hkv, u], out[:, :Hq + Hkv, v] = a * c - b * s, a * s + b * c
    return out


def attn_chunk(q, k_cache, v_cache, page_table, cu_q, seq_lens, k_scale, v_scale, sm_scale, softcap=0.0, slopes=None,
               window=0, prefix_lens=None, doc_start=None):
    """(o, a): float64 [cu_q[-1], Hq, D], a = the same with |v| (the bound of P's rounding).  Only the
    positions that a row sees enter its sums."""
    T, Hq, D = int(cu_q[-1]), q.shape[1], q.shape[2]
    P, Hkv = k_cache.shape[1], k_cache.shape[2]
    G = Hq // Hkv
    o = torch.zeros(T, Hq, D, dtype=torch.float64)
    a = torch.zeros_like(o)
    for t, (b, p) in enumerate(places(cu_q, seq_lens)):
        lo = 0 if not window else max(0, p + 1 - window)
        if doc_start is not None:
            lo = max(lo, int(doc_start[t]))
        hi = p + 1 if prefix_lens is None else max(p + 1, int(prefix_lens[b]))
        hi = min(hi, int(seq_lens[b]))
        if hi <= lo:
            continue
        j = torch.arange(lo, hi)
        page = page_table[b].long()[j // P]
        k = k_cache.view(torch.uint8)[page, j % P].view(torch.float8_e4m3fn).float().double() * k_scale.double()[:, None]
        v = v_cache.view(torch.uint8)[page, j % P].view(torch.float8_e4m3fn).float().double() * v_scale.double()[:, None]
        s = torch.einsum("hgd,lhd->hgl", q[t].double().view(Hkv, G, D), k) * sm_scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.double().view(Hkv, G, 1) * (j - p).abs().double()
        w = torch.softmax(s, -1)
        o[t] = torch.einsum("hgl,lhd->hgd", w, v).reshape(Hq, D)
        a[t] = torch.einsum("hgl,lhd->hgd", w, v.abs()).reshape(Hq, D)
    return o, a
