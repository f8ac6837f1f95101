"""Test infrastructure: plain restatements of the paged-cache operators
(bozo_b200/paged.py).  Placement and quantisation follow the definition in
fp32, one rounding per operation; attention is float64 over each sequence's own
list of cached rows."""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
TINY = 2.0 ** -100


def rotate(x, cos, sin, pos):
    """Half-split RoPE of ``x [N, heads, HD]`` at positions ``pos [N]``, in the
    tables' precision, every product and sum rounded."""
    x = x.to(cos.dtype)
    c, s = cos[pos][:, None], sin[pos][:, None]
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def quantise(x, dtype):
    """fp32 ``x [..., HD]`` → (codes, scales [...])."""
    a = x.abs().amax(-1)
    top = torch.full_like(a, TOP[dtype])  # a tensor: x / number and number / x round twice
    bad = ~torch.isfinite(a)
    tiny = a < TINY
    safe = torch.where(bad | tiny, torch.ones_like(a), a)
    most = torch.full_like(a, torch.finfo(torch.float32).max) / top
    if TOP[dtype] == 127.0:  # rounded up, where top · scale has to stay finite
        most = torch.nextafter(most, torch.zeros_like(most))
    scale = torch.minimum(safe / top, most)
    y = x * (top / safe)[..., None]
    y = torch.where((bad | tiny)[..., None], torch.zeros_like(y), y)
    scale = torch.where(tiny, torch.zeros_like(scale), scale)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    y = y.clamp(-TOP[dtype], TOP[dtype])
    return (y.round() if dtype == torch.int8 else y).to(dtype), scale


def hold(x, dtype):
    """What a page holds for fp32 rows ``x``: (rows in ``dtype``, scales or None)."""
    return quantise(x, dtype) if dtype in TOP else (x.to(dtype), None)


def place(table, b, pos, page):
    """(page number, row) of position ``pos`` of sequence b."""
    s = pos % (table.shape[1] * page)
    return int(table[b, s // page]), s % page


def attend(q, keys, values, scale, normalize):
    """One query ``q [HD]`` over ``keys, values [n, HD]`` in float64: (out, τ [n])."""
    if keys.shape[0] == 0:
        return torch.zeros_like(q), q.new_zeros(0)
    tau = torch.sigmoid(keys @ q / scale)
    out = (tau[:, None] * values).sum(0)
    if normalize == "mass":
        out = out / tau.sum().clamp(min=1e-6)
    elif normalize == "count":
        out = out / max(keys.shape[0], 1)
    return out, tau


def decode(q, hist, t, *, window, capacity, scale, normalize, tau_width):
    """``q [B, H, HD]`` (rotated, float64) against ``hist[b] = (k, v)``, each
    ``[tokens, Hk, HD]`` float64 with row s position s of the sequence.  Returns
    (out [B, H, HD], τ rows [B, H, tau_width])."""
    B, H, HD = q.shape
    out = torch.zeros(B, H, HD, dtype=torch.float64)
    tau = torch.zeros(B, H, tau_width, dtype=torch.float64)
    for b in range(B):
        if t[b] < 0:
            continue
        hi = t[b] if window else t[b] + 1
        lo = max(0, hi - (window or capacity))
        k, v = hist[b]
        G = H // k.shape[1]
        for h in range(H):
            o, row = attend(q[b, h], k[lo:hi, h // G], v[lo:hi, h // G], scale, normalize)
            out[b, h] = o
            n = row.shape[0]
            for j in range(n):          # key position lo + j
                w = tau_width - n + j if window else n - 1 - j
                if 0 <= w < tau_width:
                    tau[b, h, w] = row[j]
    return out, tau
