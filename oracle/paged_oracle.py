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


# ── 4-bit rows ──

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TINY4 = 2.0 ** -80


def hold4(x):
    """fp32 rows ``x [..., HD]`` → (codes [..., HD/2] uint8, groups [..., HD/16] e4m3,
    scales [...]).  Each quotient is one correctly rounded fp32 division."""
    a = x.abs().amax(-1)
    bad, tiny = ~torch.isfinite(a), a < TINY4
    mant, exp = torch.frexp(torch.where(bad | tiny, torch.ones_like(a), a))
    scale = torch.ldexp(torch.ones_like(a), exp - 12 + (mant > 2688 / 4096).int())
    y = torch.where((bad | tiny)[..., None], torch.zeros_like(x), x).unflatten(-1, (-1, 16))
    group = (y.abs().amax(-1) / torch.full_like(a, 6.0)[..., None]).double() / scale.double()[..., None]
    most = torch.where(scale == 2.0 ** 117, 320.0, 448.0)[..., None]
    group = torch.minimum(group, most.double()).float().to(torch.float8_e4m3fn)
    unit = group.float() * scale[..., None]
    z = torch.where(bad[..., None], torch.zeros_like(x), x).unflatten(-1, (-1, 16))
    z = z / torch.where(unit == 0, torch.full_like(unit, math.inf), unit)[..., None]
    m = z.abs()
    # to the nearest level, a tie to the one with an even number
    code = sum((m > t).int() for t in (0.25, 1.25, 2.5, 5.0)) + sum((m >= t).int() for t in (0.75, 1.75, 3.5))
    code = (code + 8 * torch.signbit(z).int()).to(torch.uint8).flatten(-2)
    scale = torch.where(tiny, torch.zeros_like(scale), scale)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    return code[..., 0::2] | code[..., 1::2] << 4, group, scale


def unhold4(codes, group, scale):
    """(code · group) · scale, the second product rounded to fp32."""
    levels = torch.tensor(LEVELS)
    levels = torch.cat([levels, -levels])
    x = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], dim=-1).flatten(-2)
    x = (x.unflatten(-1, (-1, 16)) * group.float()[..., None]).flatten(-2)
    return x * scale[..., None]


# ── page tables: plain lists, one entry at a time ──

def reserve(table, lengths, tokens, refs, page, rows):
    """(table, refs, cu, missing, places [rows] of (seq, pos, slot)) as lists."""
    table, refs = [list(r) for r in table], list(refs)
    M, P = len(table[0]), len(refs)
    wants, cu = [], [0]
    for b, t in enumerate(lengths):
        n = max(0, tokens[b]) if t >= 0 else 0
        cu.append(cu[-1] + n)
        if not n:
            continue
        cols = list(range(min(M, -(-t // page)), min(M, -(-(t + n) // page))))
        while cols and 0 <= table[b][cols[0]] < P:
            cols.pop(0)
        wants += [(b, c) for c in cols]
    free = [p for p in range(P) if refs[p] == 0]
    missing = max(0, len(wants) - len(free))
    if not missing:
        for (b, c), p in zip(wants, free):
            table[b][c], refs[p] = p, 1
    places = []
    for b in range(len(lengths)):
        for i in range(cu[b + 1] - cu[b]):
            pos, slot = lengths[b] + i, -1
            if i >= cu[b + 1] - cu[b] - M * page:
                p = table[b][pos % (M * page) // page]
                slot = p * page + pos % page if 0 <= p < P else -1
            places.append((b, pos, slot))
    places = (places + [(-1, -1, -1)] * rows)[:rows]
    return table, refs, cu, missing, places


def fork(table, lengths, parents, refs, page, share):
    """(table, refs, copies, missing) as lists."""
    M, P, R = len(table[0]), len(refs), len(table)
    refs, new, wants, seen = list(refs), [], [], set()
    copies = [(-1, -1)] * (R if share else R * M)
    for r, x in enumerate(parents):
        if not 0 <= x < R:
            new.append([-1] * M)
            continue
        t = max(0, lengths[x])
        full, held = (min(M, t // page) if share else 0), min(M, -(-t // page))
        if x in seen:
            new.append([table[x][c] if c < full else -1 for c in range(M)])
            wants += [(r, x, c) for c in range(full, held)]
        else:
            seen.add(x)
            new.append(list(table[x]))
    for rows, d in ((table, -1), (new, 1)):
        for row in rows:
            for p in row:
                if 0 <= p < P:
                    refs[p] += d
    free = [p for p in range(P) if refs[p] == 0]
    for (r, x, c), p in zip(wants, free):
        new[r][c], refs[p] = p, 1
        if 0 <= table[x][c] < P:
            copies[r if share else r * M + c] = (table[x][c], p)
    return new, refs, copies, max(0, len(wants) - len(free))


# ── beam search ──

def select(logits, scores, done, eos):
    """(scores, tokens, rows) of ``logits [N·K, V]``, in float64, by sorting every
    candidate."""
    N, K = scores.shape
    V = logits.shape[1]
    res = []
    for n in range(N):
        cand = []
        for k in range(K):
            x, s = logits[n * K + k].double(), float(scores[n, k])
            if done is not None and bool(done[n, k]):
                val = torch.full((V,), -math.inf, dtype=torch.float64)
                val[eos] = s
            else:
                m = float(x.max())
                lse = m + math.log(float(torch.exp(x - m).sum())) if math.isfinite(m) else math.nan
                val = s + (x - lse)
            if not math.isfinite(s):
                val = torch.full((V,), -math.inf, dtype=torch.float64)
            val = torch.nan_to_num(val, nan=-math.inf, posinf=-math.inf, neginf=-math.inf)
            if bool(torch.isnan(x).any()) and not (done is not None and bool(done[n, k])):
                val = torch.full((V,), -math.inf, dtype=torch.float64)
            order = torch.sort(val, descending=True, stable=True)[1][:K].tolist()
            cand += [(-float(val[v]), k, v) for v in order]
        best = sorted(cand)[:K]
        res.append(([-c[0] for c in best], [c[2] for c in best], [n * K + c[1] for c in best]))
    return (torch.tensor([r[0] for r in res], dtype=torch.float64), torch.tensor([r[1] for r in res]),
            torch.tensor([r[2] for r in res], dtype=torch.int32))
