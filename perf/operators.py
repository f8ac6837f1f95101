"""Cases of the paged-cache operators of ``bozo_b200.paged``: writing new keys
and values into a paged cache (rotated, and quantised where the cache holds 8
bits), reading them back, and the tension of one new token over the cache.

``own = False`` computes an operator in its plain form (elementary torch
operations in 32 bits, rounded once), ``own = True`` through the package's
entry points.  Both work on the same tensors:

* pages ``[P, Hk, page, HD]`` of keys (rotated) and of values, and for 8-bit
  pages one fp32 scale a row, ``[P, Hk, page]``: a row stands for code · scale;
* a page table ``[B, M]`` (int32, −1 where no page is allocated): position s of
  sequence b lies in page ``table[b, (s mod C) / page]``, row ``s mod page``,
  with ``C = M · page``, so a table narrower than a sequence is a ring;
* ``lengths [B]`` (int32): the position of each sequence's (first) new token.

8-bit rows: a = max |x|; scale = a / top, code = round(x · (top / a)), top =
448 (e4m3) or 127 (integers); a row with a < 2^-100 is held as zeros.
"""
import math
import random

import torch

own = False

_IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_STORE = dict(_IO, fp8=torch.float8_e4m3fn, int8=torch.int8)
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1, "int8": 1}
_TOP = {"fp8": 448.0, "int8": 127.0}
_TINY = 2.0 ** -100


# ── cases ──

def listed():
    return [
        # the append of a decode step of the 117M model's layer: 16 sequences, latency counts
        _write("append step 117m", B=16, Hk=12, HD=64, store="bf16", io="bf16", page=16, M=64,
               t_lo=960, t_hi=1023, new_lo=1, new_hi=1, lens=1),
        # 16 ragged prompts of the 117M model (up to its 1024 positions) entering the cache
        _write("prompts 117m", B=16, Hk=12, HD=64, store="bf16", io="bf16", page=16, M=64,
               t_lo=0, t_hi=0, new_lo=61, new_hi=1024, lens=2),
        # prompts of the 350M model's heads kept in e4m3 and read back for the next chunk
        _write("prompts to e4m3 and back", B=32, Hk=16, HD=64, store="fp8", io="bf16", page=16,
               M=160, t_lo=0, t_hi=500, new_lo=255, new_hi=2048, lens=3),
        # one token a sequence into an 8-bit integer cache, and its row back: latency counts
        _write("append step to int8 and back", B=64, Hk=16, HD=64, store="int8", io="bf16",
               page=32, M=64, t_lo=1, t_hi=2046, new_lo=1, new_hi=1, lens=4),
        # the last 64 keys of 16 sequences (a local layer's window of the 117M model)
        _read("read windows 117m", B=16, Hk=12, HD=64, store="bf16", io="bf16", page=16, M=64,
              t_lo=64, t_hi=959, new_lo=64, new_hi=64, lens=5),
        # whole long sequences out of an e4m3 cache (moving them, or attending a further chunk)
        _read("read long e4m3", B=8, Hk=16, HD=64, store="fp8", io="bf16", page=64, M=257,
              t_lo=0, t_hi=3, new_lo=4095, new_hi=16384, lens=6),
        # decode step of a local layer of the 117M model: window 64 in a ring of 5 pages, append
        _decode("window step 117m", B=16, H=12, Hk=12, HD=64, store="bf16", io="bf16", page=16,
                M=5, t_lo=200, t_hi=1000, window=64, norm="count", tau=0, append=True, lens=7),
        # decode step of a global layer of the 117M model near its 1024 positions, append
        _decode("global step 117m", B=16, H=12, Hk=12, HD=64, store="bf16", io="bf16", page=16,
                M=64, t_lo=500, t_hi=1023, window=0, norm="mass", tau=0, append=True, lens=8),
        # the 1.1M model in fp32 with its τ rows exported, windows still filling: smallest call
        _decode("window step 1m fp32 with tau", B=8, H=4, Hk=4, HD=32, store="f32", io="f32",
                page=8, M=32, t_lo=0, t_hi=255, window=64, norm="mass", tau=64, append=True,
                lens=9),
        # one very long sequence: few rows, a long axis to split
        _decode("one long sequence", B=1, H=16, Hk=16, HD=64, store="bf16", io="bf16", page=64,
                M=2048, t_lo=120001, t_hi=120001, window=0, norm="mass", tau=0, append=False,
                lens=10),
        # a serving batch of the 350M model's heads with very uneven lengths
        _decode("ragged batch", B=64, H=16, Hk=16, HD=64, store="bf16", io="bf16", page=16,
                M=512, t_lo=1, t_hi=8191, window=0, norm="mass", tau=0, append=True, lens=11),
        # long uneven sequences in an 8-bit cache whose key heads are shared by four query heads
        _decode("ragged e4m3, shared heads", B=64, H=32, Hk=8, HD=128, store="fp8", io="bf16",
                page=32, M=512, t_lo=1, t_hi=16383, window=0, norm="mass", tau=0, append=False,
                lens=12),
    ]


def _write(name, **f):
    return dict(f, name=name, op="write", H=f["Hk"])


def _read(name, **f):
    return dict(f, name=name, op="read", H=f["Hk"])


def _decode(name, **f):
    return dict(f, name=name, op="decode", new_lo=1, new_hi=1)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "decode", "decode"))
    HD = rng.choice((32, 64, 64, 64, 128))
    store = rng.choice(("bf16", "bf16", "f16", "fp8", "int8", "f32"))
    io = store if store in _IO else rng.choice(("bf16", "bf16", "f16"))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    c = dict(op=op, HD=HD, store=store, io=io, page=page, lens=rng.randrange(1 << 20))
    if op == "decode":
        Hk = rng.choice((1, 2, 4, 6, 8, 12, 16))
        H = Hk * rng.choice((1, 1, 1, 2, 4, 8))
        c.update(H=H, Hk=Hk, window=rng.choice((0, 0, rng.randint(1, 300))),
                 norm=rng.choice(("mass", "mass", "count", "none")))
        c["B"] = _log(rng, 1, 64)
        # at most about the largest listed case's keys · heads · width
        most = max(16, int(2 ** 29 / (c["B"] * Hk * HD * _SIZE[store])))
        c["t_hi"] = _log(rng, 1, min(130000, most))
        c["t_lo"] = rng.randint(0, c["t_hi"])
        c["tau"] = c["window"] or 64 if rng.random() < 0.3 else 0
        c["append"] = store in _IO and rng.random() < 0.6
        if c["window"]:
            c["M"] = -(-(c["window"] + 1) // page) + rng.randint(0, 3)
            c["norm"] = rng.choice(("mass", "count"))
        else:
            c["M"] = -(-(c["t_hi"] + 1) // page) + rng.randint(0, 2)
            c["norm"] = "none" if c["norm"] == "none" else "mass"
        return dict(c, new_lo=1, new_hi=1)
    c["Hk"] = c["H"] = rng.choice((1, 2, 4, 6, 8, 12, 16))
    c["B"] = _log(rng, 1, 128)
    most = max(1, int(2 ** 25 / (c["B"] * c["Hk"] * HD)) * 2)
    c["new_hi"] = _log(rng, 1, min(16384, most))
    c["new_lo"] = rng.randint(1, c["new_hi"])
    c["t_hi"] = rng.randint(0, 600)
    c["t_lo"] = rng.randint(0, c["t_hi"])
    c["M"] = -(-(c["t_hi"] + c["new_hi"]) // page)
    return c


def _lens(case):
    """Each sequence's position of its first new token and number of tokens: the
    ends of both ranges are among them."""
    r = random.Random(case["lens"])
    t = [r.randint(case["t_lo"], case["t_hi"]) for _ in range(case["B"])]
    n = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    t[0], n[0] = case["t_hi"], case["new_hi"]
    if case["B"] > 1:
        t[-1], n[-1] = case["t_lo"], case["new_lo"]
    return t, n


def _keys(case, t):
    """Keys that the query at position t reaches."""
    return min(t, case["window"]) if case["window"] else min(t + 1, case["M"] * case["page"])


def work(case):
    t, n = _lens(case)
    e, i, Hk, H, HD = _SIZE[case["store"]], _SIZE[case["io"]], case["Hk"], case["H"], case["HD"]
    held = HD * e + (4 if case["store"] in _TOP else 0)  # a row and its scale
    if case["op"] == "decode":
        keys = sum(_keys(case, x) for x in t)
        b = keys * Hk * 2 * held + 2 * case["B"] * H * HD * i + case["B"] * H * case["tau"] * i
        if case["append"]:
            b += case["B"] * Hk * 2 * HD * i + (case["B"] * Hk * 2 * held if case["window"] else 0)
        return {"bytes": b, "flops": 4 * keys * H * HD}
    rows = sum(n) * Hk * 2
    if case["op"] == "read":
        return {"bytes": rows * (held + HD * i), "flops": rows * HD if case["store"] in _TOP else 0}
    back = HD * i if case["store"] in _TOP else 0
    return {"bytes": rows * (HD * i + held + back) + max(n) * HD * 4,
            "flops": rows // 2 * HD * 3 + (rows * HD * 4 if back else 0)}


# ── inputs ──

def _rope_tables(HD, length, device):
    half = HD // 2
    theta = 1.0 / (10_000.0 ** (torch.arange(0, half).float() / half))
    ang = torch.outer(torch.arange(length).float(), theta)
    return ang.cos().to(device), ang.sin().to(device)


def _random_pages(case, P, g):
    """Pages as earlier tokens left them: normal rows in the cache's type (and scales)."""
    shape = (P, case["Hk"], case["page"], case["HD"])
    if case["store"] in _IO:
        return torch.randn(shape, generator=g, device="cuda", dtype=_STORE[case["store"]]), None
    return _quantise(torch.randn(shape, generator=g, device="cuda"), case["store"])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t, n = _lens(case)
    B, M, page, H, Hk, HD = (case[x] for x in ("B", "M", "page", "H", "Hk", "HD"))
    used = [min(M, -(-(a + b) // page)) for a, b in zip(t, n)]
    P = sum(used) + 3
    order = list(range(P))
    random.Random(seed).shuffle(order)
    table = [[-1] * M for _ in range(B)]
    for row, u in zip(table, used):
        for j in range(u):
            row[j] = order.pop()
    s = {"case": case, "table": torch.tensor(table, dtype=torch.int32, device="cuda"),
         "lengths": torch.tensor(t, dtype=torch.int32, device="cuda")}
    s["k_pages"], s["k_scale"] = _random_pages(case, P, g)
    s["v_pages"], s["v_scale"] = _random_pages(case, P, g)
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    s["rows"] = cu[-1]
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda") if case["op"] != "decode" else None
    s["rope"] = _rope_tables(HD, max(a + b for a, b in zip(t, n)), "cuda")
    if case["op"] != "read":
        # views of one projection's packed rows [q | k | v], as the model makes them
        x = torch.randn(cu[-1], (H + 2 * Hk) * HD, generator=g, device="cuda", dtype=_IO[case["io"]])
        q, k, v = x.split([H * HD, Hk * HD, Hk * HD], dim=-1)
        s["q"], s["k"], s["v"] = q.unflatten(1, (H, HD)), k.unflatten(1, (Hk, HD)), v.unflatten(1, (Hk, HD))
    return s


# ── one pass ──

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from bozo_b200 import paged
    c = s["case"]
    at = (s["k_pages"], s["v_pages"], s["table"], s["lengths"])
    scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "decode":
        new = (s["k"], s["v"]) if c["append"] else (None, None)
        r = paged.paged_tension(s["q"], *at, window=c["window"] or None, normalize=c["norm"],
                                rope=s["rope"], k=new[0], v=new[1], return_tau=bool(c["tau"]),
                                tau_window=c["tau"] or None, **scales)
        out = {"out": r[0], "tau": r[1]} if c["tau"] else {"out": r}
        return dict(out, k_pages=s["k_pages"], v_pages=s["v_pages"]) if c["append"] else out
    if c["op"] == "write":
        paged.write_kv(s["k"], s["v"], *at, cu_rows=s["cu"], rope=s["rope"], **scales)
        if c["store"] in _IO:
            return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    k, v = paged.read_kv(*at, s["cu"], s["rows"], dtype=_IO[c["io"]], **scales)
    return {"k": k, "v": v}


def _run_plain(s):
    c = s["case"]
    if c["op"] == "decode":
        pos = s["lengths"].long()
        seq = torch.arange(c["B"], device="cuda")
        if c["append"]:
            _put(s, seq, pos)
        out = _attend(s, pos)
        return dict(out, k_pages=s["k_pages"], v_pages=s["v_pages"]) if c["append"] else out
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["cu"], row, right=True) - 1
    pos = s["lengths"].long()[seq] + row - s["cu"].long()[seq]
    if c["op"] == "write":
        _put(s, seq, pos)
        if c["store"] in _IO:
            return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    pid, slot = _place(s, seq, pos)
    io = _IO[c["io"]]
    return {"k": _values(s["k_pages"], s["k_scale"], pid, slot).to(io),
            "v": _values(s["v_pages"], s["v_scale"], pid, slot).to(io)}


def _place(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos % (s["case"]["M"] * page) // page].long(), pos % page


def _values(pages, scale, pid, slot):
    x = pages[pid, :, slot].float()
    return x if scale is None else x * scale[pid, :, slot].unsqueeze(-1)


def _rotate(x, rope, pos):
    cos, sin = (t[pos].unsqueeze(1) for t in rope)
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _quantise(x, store):
    a = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(a, _TOP[store])  # a division by a number would be a product with its inverse
    y = torch.where(a < _TINY, 0.0, x * (top / a))
    scale = torch.where(a < _TINY, 0.0, a / top)[..., 0]
    if store == "int8":
        return y.round().clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _put(s, seq, pos):
    pid, slot = _place(s, seq, pos)
    k, v = _rotate(s["k"], s["rope"], pos), s["v"].float()
    store = s["case"]["store"]
    if store in _TOP:
        k, s["k_scale"][pid, :, slot] = _quantise(k, store)
        v, s["v_scale"][pid, :, slot] = _quantise(v, store)
    s["k_pages"][pid, :, slot] = k.to(_STORE[store])
    s["v_pages"][pid, :, slot] = v.to(_STORE[store])


def _attend(s, t):
    c = s["case"]
    B, H, Hk, HD = c["B"], c["H"], c["Hk"], c["HD"]
    most = max(1, _keys(c, c["t_hi"]))
    hi = t if c["window"] else t + 1
    n = hi.clamp(max=c["window"] or c["M"] * c["page"])
    j = torch.arange(most, device="cuda")
    live = j < n[:, None]
    pid, slot = _place(s, torch.arange(B, device="cuda")[:, None], (hi - n)[:, None] + j)
    pid = torch.where(live, pid, 0)
    k = _values(s["k_pages"], s["k_scale"], pid, slot).permute(0, 2, 3, 1)   # [B, Hk, HD, keys]
    q = _rotate(s["q"], s["rope"], t).view(B, Hk, H // Hk, HD)
    score = (q @ k) / math.sqrt(HD)
    del k
    tau = torch.where(live[:, None, None], 1 / (1 + torch.exp(-score)), 0.0)
    v = _values(s["v_pages"], s["v_scale"], pid, slot)
    v = torch.where(live[..., None, None], v, 0.0).permute(0, 2, 1, 3)       # [B, Hk, keys, HD]
    out = tau @ v
    if c["norm"] == "mass":
        out = out / tau.sum(-1, keepdim=True).clamp(min=1e-6)
    elif c["norm"] == "count":
        out = out / n.clamp(min=1).view(B, 1, 1, 1)
    io = _IO[c["io"]]
    res = {"out": out.reshape(B, H, HD).to(io)}
    if c["tau"]:
        # slot w of a window is key t − (window − w), column c of a global row key t − c
        w = torch.arange(c["tau"], device="cuda")
        col = w - c["tau"] + n[:, None] if c["window"] else n[:, None] - 1 - w
        row = tau.reshape(B, H, most).gather(
            2, col.clamp(0, most - 1)[:, None].expand(B, H, c["tau"]))
        res["tau"] = torch.where((col >= 0)[:, None], row, 0.0).to(io)
    return res


# ── from the definitions in 64 bits, one sequence at a time ──

def exact(case, seed):
    s = prepare(case, seed)
    t, n = _lens(case)
    table = s["table"].tolist()
    pages = {x: s[x + "_pages"].double() if case["store"] not in _TOP else
             s[x + "_pages"].double() * s[x + "_scale"].double()[..., None] for x in "kv"}
    angle = torch.outer(torch.arange(s["rope"][0].shape[0], device="cuda").float(),
                        (1.0 / (10_000.0 ** (torch.arange(0, case["HD"] // 2).float()
                                             / (case["HD"] // 2)))).cuda()).double()

    def turned(x, first):
        ang = angle[first:first + x.shape[0], None]
        z = torch.complex(*x.double().chunk(2, dim=-1)) * torch.polar(torch.ones_like(ang), ang)
        return torch.cat([z.real, z.imag], dim=-1)

    def where(b, first, count):
        p = torch.arange(first, first + count, device="cuda") % (case["M"] * case["page"])
        ids = torch.tensor(table[b], device="cuda")[torch.div(p, case["page"], rounding_mode="floor")]
        return ids, p % case["page"]

    def held(x):
        if case["store"] not in _TOP:
            return x
        step = x.abs().amax(-1, keepdim=True) / _TOP[case["store"]]
        if case["store"] == "int8":
            return torch.round(x / step) * step
        y = x / step
        ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / ulp) * ulp * step

    first = 0
    for b in range(case["B"] if case["op"] == "write" or case.get("append") else 0):
        at = where(b, t[b], n[b])
        rows = slice(first, first + n[b])
        pages["k"][at[0], :, at[1]] = held(turned(s["k"][rows], t[b]))
        pages["v"][at[0], :, at[1]] = held(s["v"][rows].double())
        first += n[b]
    if case["op"] != "decode":
        if case["op"] == "write" and case["store"] not in _TOP:
            return {"k_pages": pages["k"], "v_pages": pages["v"]}
        ats = [where(b, t[b], n[b]) for b in range(case["B"])]
        return {x: torch.cat([pages[x][a[0], :, a[1]] for a in ats]) for x in "kv"}
    G = case["H"] // case["Hk"]
    outs, taus = [], []
    for b in range(case["B"]):
        m = _keys(case, t[b])
        end = t[b] if case["window"] else t[b] + 1
        at = where(b, end - m, m)
        k, v = (pages[x][at[0], :, at[1]].repeat_interleave(G, dim=1) for x in "kv")
        if case["append"]:  # the new row is attended as the cache holds it
            dt = _STORE[case["store"]]
            k, v = k.to(dt).double(), v.to(dt).double()
        tau = torch.sigmoid((turned(s["q"][b:b + 1], t[b]) * k).sum(-1) / math.sqrt(case["HD"]))
        o = (tau[..., None] * v).sum(0)
        if case["norm"] == "mass":
            o = o / tau.sum(0).clamp(min=1e-6)[:, None]
        elif case["norm"] == "count":
            o = o / max(m, 1)
        outs.append(o)
        if case["tau"]:
            row = torch.zeros(case["H"], case["tau"], device="cuda", dtype=torch.float64)
            for h0 in range(0, min(m, case["tau"])):  # h0 keys back from the newest
                w = case["tau"] - 1 - h0 if case["window"] else h0
                row[:, w] = tau[m - 1 - h0]
            taus.append(row)
    res = {"out": torch.stack(outs)}
    if case["tau"]:
        res["tau"] = torch.stack(taus)
    if case["append"]:
        res.update(k_pages=pages["k"], v_pages=pages["v"])
    return res
