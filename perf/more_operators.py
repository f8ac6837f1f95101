"""Cases of decoding many hypotheses over paged caches held in 4 bits: the cache's
own operators (``bozo_b200.paged``: rows written and read back, the tension of one
new token), the page tables and row places built from request lengths
(``paged.reserve``), and beam search's selection (``beam.select``) with the
reordering of the page tables and the copies that go with it (``paged.fork``,
``paged.copy_pages``).

``own = False`` computes an operator in its plain form (elementary torch operations),
``own = True`` through the package's entry points.  Both work on the same tensors:

* 4-bit pages ``[P, Hk, page, HD/2]``: element 2i of a row in the low, 2i + 1 in the
  high four bits of byte i, as e2m1 (sign, 0 ½ 1 1½ 2 3 4 6); one e4m3 scale for 16
  elements ``[P, Hk, page, HD/16]``; one fp32 scale a row ``[P, Hk, page]``, a power
  of two.  An element stands for (e2m1 · e4m3) · fp32.  A row x is held so: scale is
  the least power of two with max |x| ≤ 6 · 448 · scale; of each sixteen, group =
  e4m3(max |x| / 6 / scale) and code = e2m1(x / (group · scale)), both to the nearest,
  ties to even; a row with max |x| < 2^-80, and sixteen whose group is 0, are zeros;
* a page table ``[B, M]`` (int32, −1 where there is no page): position s of sequence b
  lies in page ``table[b, (s mod C) / page]``, row ``s mod page``, ``C = M · page``;
* ``lengths [B]`` (int32): the position of each sequence's next token, negative where
  it is idle;
* ``refs [P]`` (int32): how many rows of the table hold a page; 0: it is free.
"""
import math
import random

import torch

own = False

_IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_TINY = 2.0 ** -80


# ── cases ──

def listed():
    return [
        # one token a sequence into a 4-bit cache of the 350M model's heads, and its row
        # back: latency counts
        _cache("append step and back", "write", B=64, H=16, Hk=16, HD=64, io="bf16", page=16, M=128,
               t_lo=1, t_hi=2046, new_lo=1, new_hi=1, lens=1),
        # ragged prompts of the same model into the cache, read back for the next chunk
        _cache("prompts and back", "write", B=32, H=16, Hk=16, HD=64, io="bf16", page=16, M=160,
               t_lo=0, t_hi=500, new_lo=255, new_hi=2048, lens=2),
        # decode step of a local layer of the 117M model: a window of 64 in a ring of 5 pages
        _cache("window step 117m", "decode", B=16, H=12, Hk=12, HD=64, io="bf16", page=16, M=5,
               t_lo=200, t_hi=1000, new_lo=1, new_hi=1, window=64, norm="count", lens=3),
        # one very long sequence: few rows, a long axis to split
        _cache("one long sequence", "decode", B=1, H=16, Hk=16, HD=64, io="bf16", page=64, M=2048,
               t_lo=120001, t_hi=120001, new_lo=1, new_hi=1, window=0, norm="mass", lens=4),
        # a serving batch of the 350M model's heads with very uneven lengths
        _cache("ragged batch", "decode", B=64, H=16, Hk=16, HD=64, io="bf16", page=16, M=512,
               t_lo=1, t_hi=8191, new_lo=1, new_hi=1, window=0, norm="mass", lens=5),
        # long uneven sequences whose key heads are shared by four query heads
        _cache("ragged, shared heads", "decode", B=64, H=32, Hk=8, HD=128, io="bf16", page=32, M=512,
               t_lo=1, t_hi=16383, new_lo=1, new_hi=1, window=0, norm="mass", lens=6),
        # the pages and row places of a decode step of 64 sequences: latency counts
        _reserve("reserve a step", B=64, page=16, M=128, t_lo=1, t_hi=2046, new_lo=1, new_hi=1,
                 spare=300, lens=7),
        # the pages and row places of a large batch of prompts
        _reserve("reserve prompts", B=256, page=16, M=160, t_lo=0, t_hi=300, new_lo=1, new_hi=2048,
                 spare=5000, lens=8),
        # a beam step's page tables and caches: the global layers of the 117M model
        _fork("fork global layers 117m", share=True, N=16, K=4, page=16, M=64, t_lo=100, t_hi=1023,
              row=2 * 12 * 64, pools=6, spare=40, lens=9),
        # and the rings of the 350M model's local layers, held in 4 bits
        _fork("fork rings 350m", share=False, N=8, K=8, page=16, M=9, t_lo=150, t_hi=2040,
              row=16 * 32, pools=32, spare=0, lens=10),
        # four hypotheses of one prompt over the 13M model's vocabulary: the smallest selection
        _select("select 1 x 4", N=1, K=4, V=8192, dtype="f32", done=False, lens=11),
        # eight hypotheses of 64 prompts over the larger models' vocabulary, some ended
        _select("select 64 x 8", N=64, K=8, V=32768, dtype="bf16", done=True, lens=12),
    ]


def _cache(name, op, **f):
    return dict(f, name=name, op=op)


def _reserve(name, **f):
    return dict(f, name=name, op="reserve")


def _fork(name, **f):
    return dict(f, name=name, op="fork")


def _select(name, **f):
    return dict(f, name=name, op="select")


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "decode", "decode", "reserve", "fork", "select"))
    c = dict(op=op, page=rng.choice((8, 16, 16, 32, 64)), lens=rng.randrange(1 << 20))
    if op == "select":
        N, K = _log(rng, 1, 128), rng.choice((1, 2, 3, 4, 5, 8, 16))
        return dict(c, N=N, K=K, V=_log(rng, 97, min(131072, 2 ** 25 // (N * K))),
                    dtype=rng.choice(("bf16", "bf16", "f16", "f32")), done=rng.random() < 0.5)
    if op == "reserve":
        c.update(B=_log(rng, 1, 512), t_hi=rng.randint(0, 3000))
        c.update(t_lo=rng.randint(0, c["t_hi"]), new_hi=_log(rng, 1, min(16384, 2 ** 18 // c["B"])))
        c["new_lo"] = rng.randint(0, min(1, c["new_hi"] - 1))
        return dict(c, M=-(-(c["t_hi"] + c["new_hi"]) // c["page"]) + rng.randint(0, 2),
                    spare=c["B"] * (-(-c["new_hi"] // c["page"]) + 1) + rng.randint(0, 100))
    if op == "fork":
        c.update(share=rng.random() < 0.6, N=_log(rng, 1, 24), K=rng.choice((1, 2, 3, 4, 8)))
        c.update(t_hi=_log(rng, 1, 1500) if c["share"] else rng.randint(1, 3000))
        c.update(t_lo=rng.randint(1, c["t_hi"]))
        if c["share"]:
            c["M"] = -(-(c["t_hi"] + 1) // c["page"]) + rng.randint(0, 2)
        else:
            c["M"] = -(-(rng.randint(4, 128) + 1) // c["page"])
        return dict(c, row=rng.choice((64, 192, 512, 768, 1536)), pools=rng.choice((2, 6, 18, 24)),
                    spare=rng.randint(0, 40))
    HD = rng.choice((32, 64, 64, 128))
    Hk = rng.choice((1, 2, 4, 6, 8, 12, 16))
    c.update(HD=HD, Hk=Hk, H=Hk, io=rng.choice(("bf16", "bf16", "f16", "f32")))
    if op == "write":
        c["B"] = _log(rng, 1, 128)
        c["new_hi"] = _log(rng, 1, max(1, min(16384, 2 ** 25 // (c["B"] * Hk * HD))))
        c.update(new_lo=rng.randint(1, c["new_hi"]), t_hi=rng.randint(0, 600))
        c["t_lo"] = rng.randint(0, c["t_hi"])
        return dict(c, M=-(-(c["t_hi"] + c["new_hi"]) // c["page"]))
    c.update(H=Hk * rng.choice((1, 1, 1, 2, 4, 8)), window=rng.choice((0, 0, rng.randint(1, 300))),
             B=_log(rng, 1, 64))
    c["t_hi"] = _log(rng, 1, min(130000, max(16, 2 ** 29 // (c["B"] * Hk * HD))))
    c["t_lo"] = rng.randint(0, c["t_hi"])
    if c["window"]:
        c.update(M=-(-(c["window"] + 1) // c["page"]) + rng.randint(0, 3),
                 norm=rng.choice(("mass", "count")))
    else:
        c.update(M=-(-(c["t_hi"] + 1) // c["page"]) + rng.randint(0, 2), norm="mass")
    return dict(c, new_lo=1, new_hi=1)


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


def _beams(case):
    """Lengths of the N prompts' hypotheses and the row that each of the next N·K
    comes from: good hypotheses have several continuations, others none."""
    r = random.Random(case["lens"])
    N, K = case["N"], case["K"]
    t = [r.randint(case["t_lo"], case["t_hi"]) for _ in range(N)]
    t[0], t[-1] = case["t_lo"], case["t_hi"]
    weight = [2.0 ** -i for i in range(K)]
    return t, [n * K + k for n in range(N) for k in r.choices(range(K), weight, k=K)]


def _keys(case, t):
    """Keys that the query at position t reaches."""
    return min(t, case["window"]) if case["window"] else min(t + 1, case["M"] * case["page"])


def _pages(case, t):
    return min(case["M"], -(-t // case["page"]))


def work(case):
    op = case["op"]
    if op == "select":
        R = case["N"] * case["K"]
        live = R if not case["done"] else R - R // case["K"]  # ended ones' logits are not read
        e = _SIZE[case["dtype"]]
        return {"bytes": live * case["V"] * e + R * 21, "flops": 4 * live * case["V"]}
    if op == "reserve":
        t, n = _lens(case)
        new = sum(_pages(case, a + b) - _pages(case, a) for a, b in zip(t, n))
        return {"bytes": 12 * case["B"] + 12 * sum(n) + 12 * new, "flops": 0}
    if op == "fork":
        t, parents = _beams(case)
        R, K, page = case["N"] * case["K"], case["K"], case["page"]
        more = [r for r in range(R) if r != parents.index(parents[r])]  # not the first of their row
        copied = sum(1 if case["share"] and t[r // K] % page else 0 if case["share"] else _pages(case, t[r // K])
                     for r in more)
        held = sum(_pages(case, t[r // K]) for r in range(R))
        return {"bytes": 8 * held + 12 * R + 2 * copied * page * case["row"] * case["pools"], "flops": 0}
    t, n = _lens(case)
    i, Hk, H, HD = _SIZE[case["io"]], case["Hk"], case["H"], case["HD"]
    held = HD // 2 + HD // 16 + 4  # a row, its group scales and its scale
    if op == "decode":
        keys = sum(_keys(case, x) for x in t)
        return {"bytes": keys * Hk * 2 * held + 2 * case["B"] * H * HD * i, "flops": 4 * keys * H * HD}
    rows = sum(n) * Hk * 2
    return {"bytes": rows * (2 * HD * i + held) + max(n) * HD * 4, "flops": rows // 2 * HD * 3 + rows * HD * 6}


# ── inputs ──

def _rope_tables(HD, length, device):
    half = HD // 2
    theta = 1.0 / (10_000.0 ** (torch.arange(0, half).float() / half))
    ang = torch.outer(torch.arange(length).float(), theta)
    return ang.cos().to(device), ang.sin().to(device)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(case, held, seed):
    """A shuffled pool and the page table whose row b holds held[b] pages."""
    P = max(1, sum(held) + case.get("spare", 3))
    order = list(range(P))
    random.Random(seed).shuffle(order)
    table, refs = [[-1] * case["M"] for _ in held], [0] * P
    for row, u in zip(table, held):
        for j in range(u):
            row[j] = order.pop()
            refs[row[j]] += 1
    return table, refs


def _random_pages(case, P, g):
    """Pages as earlier tokens left them: normal rows, held in 4 bits."""
    shape = (P, case["Hk"], case["page"], case["HD"])
    codes = torch.empty(*shape[:3], shape[3] // 2, dtype=torch.uint8, device="cuda")
    group = torch.empty(*shape[:3], shape[3] // 16, dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(shape[:3], device="cuda")
    step = max(1, 2 ** 25 // (shape[1] * shape[2] * shape[3]))
    for i in range(0, P, step):
        x = torch.randn(min(step, P - i), *shape[1:], generator=g, device="cuda")
        codes[i:i + step], group[i:i + step], scale[i:i + step] = _hold(x)
    return codes, group, scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "select":
        N, K, V = case["N"], case["K"], case["V"]
        s["logits"] = (torch.randn(N * K, V, generator=g, device="cuda") * 3).to(_IO[case["dtype"]])
        s["scores"] = -20 * torch.rand(N, K, generator=g, device="cuda")
        s["done"], s["eos"] = None, None
        if case["done"]:  # one in K has ended
            s["eos"] = V // 3
            s["done"] = torch.zeros(N, K, dtype=torch.bool, device="cuda")
            s["done"].view(-1)[K - 1::K] = True
        return s
    if op == "fork":
        t, parents = _beams(case)
        K, P0 = case["K"], 0
        held = [_pages(case, x) for x in t for _ in range(K)]
        table, refs = _tables(case, held, seed)
        if case["share"]:  # the hypotheses of a prompt share the pages of its first half
            for n, x in enumerate(t):
                for j in range(x // 2 // case["page"]):
                    refs[table[n * K][j]] = K
                    for k in range(1, K):
                        refs[table[n * K + k][j]] = 0
                        table[n * K + k][j] = table[n * K][j]
        s.update(table=_int32(table), refs=_int32(refs), parents=_int32(parents),
                 lengths=_int32([x for x in t for _ in range(K)]))
        shape = (len(refs), case["page"], case["row"])
        s["pools"] = [torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
                      for _ in range(case["pools"])]
        return s
    t, n = _lens(case)
    B, H, Hk, HD = (case.get(x) for x in ("B", "H", "Hk", "HD"))
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    s.update(lengths=_int32(t), rows=cu[-1])
    if op == "reserve":
        table, refs = _tables(case, [_pages(case, x) for x in t], seed)
        s.update(table=_int32(table), refs=_int32(refs), tokens=_int32(n))
        return s
    table, refs = _tables(case, [_pages(case, a + b) for a, b in zip(t, n)], seed)
    s["table"] = _int32(table)
    s["k_pages"], s["k_group"], s["k_scale"] = _random_pages(case, len(refs), g)
    s["v_pages"], s["v_group"], s["v_scale"] = _random_pages(case, len(refs), g)
    s["cu"] = _int32(cu) if op != "decode" else None
    s["rope"] = _rope_tables(HD, max(a + b for a, b in zip(t, n)), "cuda")
    # views of one projection's packed rows [q | k | v], as the model makes them
    x = torch.randn(cu[-1], (H + 2 * Hk) * HD, generator=g, device="cuda", dtype=_IO[case["io"]])
    q, k, v = x.split([H * HD, Hk * HD, Hk * HD], dim=-1)
    s["q"], s["k"], s["v"] = q.unflatten(1, (H, HD)), k.unflatten(1, (Hk, HD)), v.unflatten(1, (Hk, HD))
    return s


# ── one pass ──

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from bozo_b200 import beam, paged
    c = s["case"]
    if c["op"] == "select":
        scores, tokens, rows = beam.select(s["logits"], s["scores"], done=s["done"], eos=s["eos"])
        return {"scores": scores, "tokens": tokens, "rows": rows}
    if c["op"] == "reserve":
        table, refs = s["table"].clone(), s["refs"].clone()  # both are updated in place
        plan = paged.reserve(table, s["lengths"], s["tokens"], refs, c["page"], rows=s["rows"])
        return {"table": table, "refs": refs, "cu": plan.cu_rows, "missing": plan.missing,
                "seq": plan.seq, "pos": plan.pos, "slot": plan.slot}
    if c["op"] == "fork":
        table, refs = s["table"].clone(), s["refs"].clone()
        copies, missing = paged.fork(table, s["lengths"], s["parents"], refs, c["page"], share=c["share"])
        paged.copy_pages(s["pools"], copies)
        return {"table": table, "refs": refs, "copies": copies, "missing": missing, "pools": s["pools"]}
    at = (s["k_pages"].view(torch.float4_e2m1fn_x2), s["v_pages"].view(torch.float4_e2m1fn_x2),
          s["table"], s["lengths"])
    scales = {x: s[x] for x in ("k_scale", "v_scale", "k_group", "v_group")}
    if c["op"] == "decode":
        return {"out": paged.paged_tension(s["q"], *at, window=c["window"] or None, normalize=c["norm"],
                                           rope=s["rope"], **scales)}
    paged.write_kv(s["k"], s["v"], *at, cu_rows=s["cu"], rope=s["rope"], **scales)
    k, v = paged.read_kv(*at, s["cu"], s["rows"], dtype=_IO[c["io"]], **scales)
    return {"k": k, "v": v}


def _run_plain(s):
    c = s["case"]
    if c["op"] == "select":
        return _plain_select(s)
    if c["op"] == "reserve":
        return _plain_reserve(s)
    if c["op"] == "fork":
        return _plain_fork(s)
    if c["op"] == "decode":
        return _attend(s, s["lengths"].long())
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["cu"], row, right=True) - 1
    pos = s["lengths"].long()[seq] + row - s["cu"].long()[seq]
    pid, slot = _place(s, seq, pos)
    for x, new in (("k", _rotate(s["k"], s["rope"], pos)), ("v", s["v"].float())):
        codes, group, scale = _hold(new)
        s[x + "_pages"][pid, :, slot] = codes
        s[x + "_group"].view(torch.uint8)[pid, :, slot] = group.view(torch.uint8)
        s[x + "_scale"][pid, :, slot] = scale
    io = _IO[c["io"]]
    return {"k": _values(s, "k", pid, slot).to(io), "v": _values(s, "v", pid, slot).to(io)}


def _hold(x):
    """fp32 rows ``[..., HD]`` as (codes, group scales, scales)."""
    a = x.abs().amax(-1)
    tiny = a < _TINY
    m, e = torch.frexp(torch.where(tiny, 1.0, a))  # a = m · 2^e, m in [½, 1); 2688 = 0.65625 · 2^12
    scale = torch.ldexp(torch.ones_like(a), e - 12 + (m > 0.65625).int())
    y = x.unflatten(-1, (-1, 16))
    top = y.abs().amax(-1)
    group = torch.where(tiny.unsqueeze(-1), 0.0, top / torch.full_like(top, 6.0) / scale.unsqueeze(-1))
    group = group.clamp(max=448.0).to(torch.float8_e4m3fn)
    scale = torch.where(tiny, 0.0, scale)
    unit = group.float() * scale.unsqueeze(-1)
    y = y / torch.where(unit == 0, math.inf, unit).unsqueeze(-1)
    z = y.abs()
    code = ((z > 0.25).to(torch.uint8) + (z >= 0.75) + (z > 1.25) + (z >= 1.75) + (z > 2.5) + (z >= 3.5) + (z > 5))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, group, scale


def _values(s, x, pid, slot):
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    levels = torch.cat([levels, -levels])
    codes = s[x + "_pages"][pid, :, slot]
    y = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], dim=-1).flatten(-2)
    group = s[x + "_group"].view(torch.uint8)[pid, :, slot].view(torch.float8_e4m3fn).float()
    y = (y.unflatten(-1, (-1, 16)) * group.unsqueeze(-1)).flatten(-2)
    return y * s[x + "_scale"][pid, :, slot].unsqueeze(-1)


def _place(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos % (s["case"]["M"] * page) // page].long(), pos % page


def _rotate(x, rope, pos):
    cos, sin = (t[pos].unsqueeze(1) for t in rope)
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


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
    out = torch.empty(B, H, HD, device="cuda")
    group = max(1, 2 ** 28 // (most * Hk * HD))  # sequences at a time
    for b in range(0, B, group):
        e = slice(b, b + group)
        k = _values(s, "k", pid[e], slot[e]).permute(0, 2, 3, 1)             # [B, Hk, HD, keys]
        q = _rotate(s["q"][e], s["rope"], t[e]).unflatten(1, (Hk, H // Hk))
        tau = 1 / (1 + torch.exp(-(q @ k) / math.sqrt(HD)))
        del k
        tau = torch.where(live[e, None, None], tau, 0.0)
        v = _values(s, "v", pid[e], slot[e])
        v = torch.where(live[e, :, None, None], v, 0.0).permute(0, 2, 1, 3)  # [B, Hk, keys, HD]
        o = tau @ v
        if c["norm"] == "mass":
            o = o / tau.sum(-1, keepdim=True).clamp(min=1e-6)
        elif c["norm"] == "count":
            o = o / n[e].clamp(min=1).view(-1, 1, 1, 1)
        out[e] = o.flatten(1, 2)
    return {"out": out.to(_IO[c["io"]])}


def _plain_reserve(s):
    """Every sequence's table row gets pages for its new tokens, the free ones in
    ascending order, or none does where they are too few; row n of the packed new
    tokens is position ``pos`` of sequence ``seq``, at ``slot`` = page · size + row."""
    c = s["case"]
    page, M = c["page"], c["M"]
    table, refs, N = s["table"].clone(), s["refs"].clone(), s["rows"]
    P = refs.shape[0]
    t = s["lengths"].long()
    n = torch.where(t >= 0, s["tokens"].long().clamp(min=0), 0)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    col = torch.arange(M, device="cuda")
    have = ((t + page - 1) // page).clamp(0, M)
    need = torch.where(n > 0, ((t + n + page - 1) // page).clamp(0, M), have)
    hole = (col >= have[:, None]) & (col < need[:, None]) & ((table < 0) | (table >= P))
    first = torch.where(hole, col, need[:, None]).amin(1)
    want = need - first
    off = want.cumsum(0) - want
    free = refs == 0
    order = torch.sort((~free).int(), stable=True)[1]
    missing = (want.sum() - free.sum()).clamp(min=0)
    ok = missing == 0
    fresh = (col >= first[:, None]) & (col < need[:, None]) & ok
    rank = (off[:, None] + col - first[:, None]).clamp(0, P - 1)
    table = torch.where(fresh, order[rank].int(), table)
    refs = torch.where(free & (free.cumsum(0) <= want.sum()) & ok, 1, refs)
    row = torch.arange(N, device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    real = seq < c["B"]
    seq = seq.clamp(max=c["B"] - 1)
    pos = t[seq] + row - cu[seq]
    pid = table[seq, pos % (M * page) // page].long()
    kept = real & (pid >= 0) & (pid < P) & (pos >= t[seq] + n[seq] - M * page)
    slot = torch.where(kept, pid * page + pos % page, -1)
    return {"table": table, "refs": refs.int(), "cu": cu.int(), "missing": missing.int().view(1),
            "seq": torch.where(real, seq, -1).int(), "pos": torch.where(real, pos, -1).int(), "slot": slot.int()}


def _plain_fork(s):
    """Row r of the table becomes its parent's.  Where pages are shared, full ones are
    held by all children; the page that is being filled (rings: every page) stays with
    the parent's first child, and each further one gets a free page to copy it to."""
    c = s["case"]
    page, M, share = c["page"], c["M"], c["share"]
    table, refs = s["table"], s["refs"].long()
    R, P = table.shape[0], refs.shape[0]
    t, parent = s["lengths"].long(), s["parents"].long()
    row, col = torch.arange(R, device="cuda"), torch.arange(M, device="cuda")
    children = torch.zeros(R, dtype=torch.long, device="cuda").index_add_(0, parent, torch.ones_like(parent))
    eldest = torch.full((R,), R, device="cuda").scatter_reduce_(0, parent, row, "amin")
    heir = eldest[parent] == row
    full = (t // page).clamp(0, M) if share else torch.zeros_like(t)
    held = ((t + page - 1) // page).clamp(0, M)
    shared = col < full[:, None]
    real = (table >= 0) & (table < P)
    delta = torch.where(shared, children[:, None] - 1, children[:, None].clamp(max=1) - 1)
    refs = refs.index_add(0, torch.where(real, table, 0).long().view(-1), torch.where(real, delta, 0).view(-1))
    old = table[parent]
    fresh = ~heir[:, None] & (col >= full[parent][:, None]) & (col < held[parent][:, None])
    rank = fresh.view(-1).cumsum(0) - 1
    free = refs == 0
    order = torch.sort((~free).int(), stable=True)[1]
    there = fresh.view(-1) & (rank < free.sum())
    new = torch.where(there, order[rank.clamp(0, P - 1)], -1).view(R, M)
    keep = heir[:, None] | shared[parent]
    res = torch.where(keep, old, torch.where(fresh, new, -1)).int()
    refs = torch.where(free & (free.cumsum(0) <= fresh.sum()), 1, refs)
    src = torch.where(there.view(R, M) & real[parent], old, -1)
    dst = torch.where(there, new.view(-1), -1).view(R, M).int()
    if share:  # one page a row
        src, dst = src.amax(1), dst.amax(1)
    copies = torch.stack([src.reshape(-1), dst.reshape(-1)], dim=-1)
    do = (copies >= 0).all(1)
    a, b = copies[do].long().unbind(1)
    for p in s["pools"]:
        p[b] = p[a]
    missing = (fresh.sum() - free.sum()).clamp(min=0).int().view(1)
    return {"table": res, "refs": refs.int(), "copies": copies.int(), "missing": missing, "pools": s["pools"]}


def _plain_select(s):
    """The K best continuations of each prompt's K hypotheses: a hypothesis' score plus
    its token's log probability (in 64 bits: near candidates are told apart); an ended
    one goes on as itself."""
    c = s["case"]
    N, K, V = c["N"], c["K"], c["V"]
    x = s["logits"].double()
    m = x.amax(-1, keepdim=True)
    logp = x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    cand = s["scores"].double().view(N * K, 1) + logp
    if s["done"] is not None:
        end = torch.arange(V, device="cuda") == s["eos"]
        stay = torch.where(end, s["scores"].double().view(N * K, 1), -math.inf)
        cand = torch.where(s["done"].view(N * K, 1), stay, cand)
    best, at = torch.sort(cand.view(N, K * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    base = torch.arange(N, device="cuda")[:, None] * K
    return {"scores": best.float(), "tokens": at % V, "rows": (base + at // V).int()}


# ── from the definitions in 64 bits ──

def exact(case, seed):
    op = case["op"]
    if op in ("reserve", "fork"):
        return None  # whole numbers and bytes
    s = prepare(case, seed)
    if op == "select":
        logp = torch.log_softmax(s["logits"].double(), dim=-1).view(case["N"], case["K"], -1)
        if s["done"] is not None:
            logp[s["done"]] = -math.inf
            logp[..., s["eos"]] = torch.where(s["done"], 0.0, logp[..., s["eos"]])
        best = (s["scores"].double()[..., None] + logp).flatten(1).topk(case["K"]).values
        return {"scores": best, "tokens": None, "rows": None}
    t, n = _lens(case)
    angle = torch.outer(torch.arange(s["rope"][0].shape[0], device="cuda").float(),
                        (1.0 / (10_000.0 ** (torch.arange(0, case["HD"] // 2).float()
                                             / (case["HD"] // 2)))).cuda()).double()

    def turned(x, first):
        ang = angle[first:first + x.shape[0], None]
        z = torch.complex(*x.double().chunk(2, dim=-1)) * torch.polar(torch.ones_like(ang), ang)
        return torch.cat([z.real, z.imag], dim=-1)

    if op == "write":
        def held(x):
            y = x.unflatten(-1, (-1, 16))
            unit = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 2688))).unsqueeze(-1)
            g = y.abs().amax(-1, keepdim=True) / (6 * unit)
            ulp = torch.exp2(torch.floor(torch.log2(g.clamp(min=2.0 ** -6))) - 3)
            u = torch.round(g / ulp) * ulp * unit
            z = torch.where(u > 0, y / u, 0.0)
            ulp = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=1.0))) - 1)
            return ((torch.round(z / ulp) * ulp).clamp(-6, 6) * u).flatten(-2)

        ks, first = [], 0
        for a, b in zip(t, n):
            ks.append(held(turned(s["k"][first:first + b], a)))
            first += b
        return {"k": torch.cat(ks), "v": held(s["v"].double())}
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    table, page, outs = s["table"].tolist(), case["page"], []
    G = case["H"] // case["Hk"]
    for b in range(case["B"]):
        m = _keys(case, t[b])
        end = t[b] if case["window"] else t[b] + 1
        p = torch.arange(end - m, end, device="cuda") % (case["M"] * page)
        ids, row = torch.tensor(table[b], device="cuda")[torch.div(p, page, rounding_mode="floor")], p % page
        kv = []
        for x in "kv":
            byte = s[x + "_pages"][ids, :, row].int()
            code = torch.stack([byte % 16, torch.div(byte, 16, rounding_mode="floor")], -1).flatten(-2)
            val = level[code % 8] * (1 - 2 * torch.div(code, 8, rounding_mode="floor"))
            grp = s[x + "_group"].view(torch.uint8)[ids, :, row].view(torch.float8_e4m3fn).double()
            unit = grp * s[x + "_scale"][ids, :, row].double()[..., None]
            kv.append((val * unit.repeat_interleave(16, dim=-1)).permute(1, 0, 2))  # [Hk, keys, HD]
        q = turned(s["q"][b:b + 1], t[b])[0].view(case["Hk"], G, case["HD"])
        tau = torch.sigmoid(torch.einsum("hgd,hkd->hgk", q, kv[0]) / math.sqrt(case["HD"]))
        o = torch.einsum("hgk,hkd->hgd", tau, kv[1]).reshape(case["H"], case["HD"])
        if case["norm"] == "mass":
            o = o / tau.sum(-1).reshape(-1, 1).clamp(min=1e-6)
        elif case["norm"] == "count":
            o = o / max(m, 1)
        outs.append(o)
    return {"out": torch.stack(outs)}
