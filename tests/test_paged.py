"""Paged caches (``bozo_b200.paged``): ``write_kv``, ``read_kv``, ``paged_tension``.

* Writing equals the plain fp32 definition bit for bit (pages, codes, scales),
  and touches nothing else: it rounds each operation as the definition does.
* Reading equals code · scale, rounded once, bit for bit.
* The decode step is compared with a float64 restatement over each sequence's
  own list of rows.  Its sums are held in fp32 and its result is rounded once:
  |err| ≤ u·|ref| + 1e-5·max|v|, u one unit in the last place of the result's
  type (2^-7 · ½ for bf16, 2^-10 · ½ for fp16, both doubled; 1e-5 for fp32: an
  HD-long fp32 dot and an n-long sum of positive weights), τ alike with
  max|v| = 1.
* Pools start out full of NaN, so a row read out of reach shows.
"""
import math

import pytest
import torch

from bozo_b200 import _capi, ops, paged
from oracle import paged_oracle as orc

F8, I8 = torch.float8_e4m3fn, torch.int8
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ULP = {F32: 1e-5, BF16: 2.0 ** -7, F16: 2.0 ** -10}
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def rope(HD, length, device):
    return ops.rope_tables(HD, length, 10_000.0, device)


class Pool:
    """A pool of shuffled pages with the tables of B sequences, on the GPU."""

    def __init__(self, B, Hk, HD, page, width, dtype, spare=2, device="cuda", allocate=None):
        P = B * width + spare
        order = torch.randperm(P, generator=torch.Generator().manual_seed(P)).int()
        self.table = order[:B * width].view(B, width).clone()
        if allocate is not None:  # only the first pages of each sequence
            for b, n in enumerate(allocate):
                self.table[b, n:] = -1
        self.table = self.table.to(device)
        shape = (P, Hk, page, HD)
        self.k, self.v = (torch.full(shape, 0.0, device=device).to(dtype) for _ in "kv")
        self.ks = self.vs = None
        if dtype in orc.TOP:
            self.ks, self.vs = (torch.full(shape[:3], math.nan, device=device) for _ in "kv")
        else:
            self.k.fill_(math.nan), self.v.fill_(math.nan)
        self.page, self.width, self.cap, self.dtype = page, width, page * width, dtype

    @property
    def scales(self):
        return {"k_scale": self.ks, "v_scale": self.vs}

    @property
    def cache(self):
        return self.k, self.v, self.table


def bits(x):
    return x.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]).cpu()


def same_bits(a, b, what):
    assert a.dtype == b.dtype and a.shape == b.shape, what
    x, y = bits(a), bits(b)
    if a.is_floating_point() and a.element_size() > 1:  # NaN payloads may differ
        nan = torch.isnan(a.cpu())
        assert torch.equal(nan, torch.isnan(b.cpu())), what
        x, y = x.masked_fill(nan, 0), y.masked_fill(nan, 0)
    assert torch.equal(x, y), f"{what}: {int((x != y).sum())} of {x.numel()} differ"


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def plain_write(pool, k, v, start, counts, tables):
    """The pages and scales after the write, by the definition (on the CPU)."""
    res = [x.cpu().clone() if x is not None else None for x in (pool.k, pool.v, pool.ks, pool.vs)]
    pos = torch.cat([torch.arange(n) + max(s, 0) for s, n in zip(start, counts)] + [torch.zeros(0, dtype=torch.long)])
    k, v = k.cpu().float()[:len(pos)], v.cpu().float()[:len(pos)]
    if tables is not None:
        k = orc.rotate(k, tables[0].cpu(), tables[1].cpu(), pos)
    (k, ks), (v, vs) = orc.hold(k, pool.dtype), orc.hold(v, pool.dtype)
    row = 0
    for b, (s, n) in enumerate(zip(start, counts)):
        for i in range(n):
            if s >= 0 and i >= n - pool.cap:
                pid, slot = orc.place(pool.table.cpu(), b, s + i, pool.page)
                res[0][pid, :, slot], res[1][pid, :, slot] = k[row], v[row]
                if ks is not None:
                    res[2][pid, :, slot], res[3][pid, :, slot] = ks[row], vs[row]
            row += 1
    return res


def check_write(pool, k, v, start, counts, tables, cu=True):
    want = plain_write(pool, k, v, start, counts, tables)
    paged.write_kv(k, v, *pool.cache, int32(start), cu_rows=int32(offsets(counts)) if cu else None,
                   rope=tables, **pool.scales)
    for got, ref, name in zip((pool.k, pool.v, pool.ks, pool.vs), want,
                              ("k_pages", "v_pages", "k_scale", "v_scale")):
        if got is not None:
            same_bits(got.cpu(), ref, name)


# ── writing ──

@gpu
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F8, I8])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 7), (128, 8), (48, 1), (20, 5)])
def test_write_prompts_bit_for_bit(dtype, io, HD, page):
    counts, start = [19, 0, 1, 40, 7], [0, 3, 11, 5, 2]
    pool = Pool(5, 3, HD, page, -(-48 // page), dtype)
    g = torch.Generator("cuda").manual_seed(HD)
    x = torch.randn(sum(counts) + 3, 3 * 3 * HD, generator=g, device="cuda").to(io)  # 3 rows of padding
    _, k, v = (y.unflatten(1, (3, HD)) for y in x.chunk(3, dim=1))
    check_write(pool, k, v, start, counts, rope(HD, 64, "cuda"))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F8])
def test_write_one_row_a_sequence_skips_inactive_ones(dtype):
    start = [0, -1, 15, 16, 31, 100]
    pool = Pool(6, 4, 64, 16, 2, dtype)  # 100: the ring has wrapped
    k, v = (torch.randn(6, 4, 64, device="cuda", dtype=BF16) for _ in "kv")
    check_write(pool, k, v, start, [1] * 6, rope(64, 128, "cuda"), cu=False)


@gpu
@pytest.mark.parametrize("dtype", [F32, I8])
def test_write_longer_than_the_ring_keeps_its_end(dtype):
    """More tokens than the ring holds in one call: the last C, in any order of blocks."""
    pool = Pool(2, 2, 32, 8, 3, dtype)
    k, v = (torch.randn(130, 2, 32, device="cuda") for _ in "kv")
    check_write(pool, k, v, [5, 0], [100, 30], rope(32, 128, "cuda"))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F8, I8])
def test_write_strided_inputs_and_no_rope(dtype):
    """Element strides over one, heads before rows, k and v of different types."""
    k = torch.randn(4, 23, 128, device="cuda")[:, :, ::2].transpose(0, 1)
    v = torch.randn(64, 23, 4, device="cuda", dtype=F16).permute(1, 2, 0)
    pool = Pool(1, 4, 64, 16, 2, dtype)
    check_write(pool, k, v, [2], [23], None)


@gpu
@pytest.mark.parametrize("HD", [64, 40])
@pytest.mark.parametrize("dtype", [F8, I8])
def test_write_rows_that_are_hard_to_quantise(dtype, HD):
    """Zeros, one non-zero element, halfway codes, the flush limit and its
    neighbours, the largest and denormal numbers, infinities and NaN."""
    inf, top = math.inf, orc.TOP[dtype]
    rows = torch.zeros(14, 1, HD)
    rows[1, 0, 3] = -7.5
    rows[2, 0, :] = torch.arange(HD) % 32 + 0.5
    rows[2, 0, 0] = top                      # a = top: the codes are the rounded values themselves
    rows[3, 0, 5] = 2.0 ** -100
    rows[4, 0, 5] = 2.0 ** -100 * (1 - 2.0 ** -24)
    rows[5, 0, :] = 1e-41
    rows[6] = (torch.rand(1, HD) * 2 - 1) * 3e38  # finite, near the largest
    rows[7, 0, 1], rows[7, 0, 2] = torch.finfo(F32).max, 1e-30
    rows[8, 0, 9] = inf
    rows[9, 0, 9] = -inf
    rows[10, 0, 9] = math.nan
    rows[11, 0, 0], rows[11, 0, HD - 1] = math.nan, inf
    rows[12, 0, ::2] = -0.0
    rows[13] = torch.randn(1, HD)
    pool = Pool(1, 1, HD, 16, 1, dtype)
    check_write(pool, rows.cuda(), rows.flip(0).cuda(), [0], [14], None)
    k, v = paged.read_kv(*pool.cache, int32([0]), int32([0, 14]), 14, dtype=F32, **pool.scales)
    for i in (8, 9, 10, 11):
        assert torch.isnan(k[i]).all() and torch.isnan(v[13 - i]).all()
    assert (k[[0, 4, 5]] == 0).all() and torch.isfinite(k[[0, 1, 2, 3, 4, 5, 6, 7, 12, 13]]).all()


# ── reading ──

@gpu
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F8, I8])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 3), (128, 8), (20, 5)])
def test_read_bit_for_bit(dtype, out, HD, page):
    counts, start = [33, 1, 0, 12], [0, 20, 4, -1]
    pool = Pool(4, 3, HD, page, -(-48 // page), dtype)
    g = torch.Generator("cuda").manual_seed(page)
    x = torch.randn(pool.k.shape, generator=g, device="cuda")
    for name, mul in (("k", 1.0), ("v", 30.0)):
        held, scale = orc.hold(x * mul, dtype)
        getattr(pool, name).copy_(held)
        if scale is not None:
            getattr(pool, name + "s").copy_(scale)
    rows = sum(counts) + 2
    got = paged.read_kv(*pool.cache, int32(start), int32(offsets(counts)), rows, dtype=out, **pool.scales)
    for y, held, scale in zip(got, (pool.k, pool.v), (pool.ks, pool.vs)):
        ref = torch.zeros(rows, 3, HD)
        n = 0
        for b, (s, c) in enumerate(zip(start, counts)):
            for i in range(c):
                if s >= 0:
                    pid, slot = orc.place(pool.table.cpu(), b, s + i, page)
                    r = held[pid, :, slot].float()
                    ref[n] = (r if scale is None else r * scale[pid, :, slot][:, None]).cpu()
                n += 1
        same_bits(y.cpu(), ref.to(out), f"{dtype} → {out}")


# ── the decode step ──

def fill(pool, lengths, Hk, HD, io, tables, seed, scale_k=1.0):
    """Random histories written through ``write_kv``; returns hist[b] = (k, v) as
    held, float64 [tokens, Hk, HD]."""
    counts = [max(n, 0) for n in lengths]
    g = torch.Generator("cuda").manual_seed(seed)
    k, v = (torch.randn(sum(counts), Hk, HD, generator=g, device="cuda") for _ in "kv")
    k, v = (k * scale_k).to(io), v.to(io)
    zero = int32([0] * len(counts))
    paged.write_kv(k, v, *pool.cache, zero, cu_rows=int32(offsets(counts)), rope=tables, **pool.scales)
    return history(pool, counts, Hk, HD)


def history(pool, counts, Hk, HD):
    hist = []
    for b, n in enumerate(counts):
        k, v = (torch.zeros(n, Hk, HD, dtype=torch.float64) for _ in "kv")
        lo = max(0, n - pool.cap)
        if n:
            one = (pool.k, pool.v, pool.table[b:b + 1])
            x, y = paged.read_kv(*one, int32([lo]), int32([0, n - lo]), n - lo, dtype=F32, **pool.scales)
            k[lo:], v[lo:] = x.double().cpu(), y.double().cpu()
        hist.append((k, v))
    return hist


def check_decode(pool, lengths, hist, q, *, window, normalize="mass", tables=None, tau_window=None,
                 new=None, scale=None, tau=True):
    """``hist`` holds the rows before the step, and with ``new`` the step writes one more."""
    B, H, HD = q.shape
    tw = (window or tau_window) if tau else 0
    res = paged.paged_tension(q, *pool.cache, int32(lengths), window=window, normalize=normalize,
                              rope=tables, k=new[0] if new else None, v=new[1] if new else None,
                              scale=scale, return_tau=tau, tau_window=tw or None, **pool.scales)
    out, row = res if tau else (res, None)
    if new:
        hist = history(pool, [t + 1 if t >= 0 else 0 for t in lengths], pool.k.shape[1], HD)
    qr = q.cpu().double()
    if tables is not None:
        pos = torch.tensor([max(t, 0) for t in lengths])
        qr = orc.rotate(qr, tables[0].cpu().double(), tables[1].cpu().double(), pos)
    ref, ref_tau = orc.decode(qr, hist, lengths, window=window, capacity=pool.cap,
                              scale=scale or math.sqrt(HD), normalize=normalize, tau_width=tw)
    big = max([1.0] + [float(torch.nan_to_num(v).abs().max()) for _, v in hist if v.numel()])
    if normalize == "none" or normalize is None:
        big *= max(1, max(lengths))
    for got, want, unit, name in ((out, ref, big, "out"), (row, ref_tau, 1.0, "tau")):
        if got is None:
            continue
        assert got.dtype == q.dtype
        err = (got.cpu().double() - want).abs()
        bound = ULP[q.dtype] * want.abs() + 1e-5 * unit
        assert torch.isfinite(got).all(), name
        assert bool((err <= bound).all()), f"{name}: worst {float((err / bound).max()):.2f} of the bound"
    return out, row


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, -1, 200]


@gpu
@pytest.mark.parametrize("dtype,io", [(F32, F32), (BF16, BF16), (F16, F16), (F8, BF16), (I8, F16),
                                      (BF16, F32), (F8, F32)])
@pytest.mark.parametrize("HD", [32, 64, 128, 48])
@pytest.mark.parametrize("window,normalize", [(16, "mass"), (64, "count"), (1, "none"), (None, "mass"),
                                              (None, None)])
def test_decode_matches_float64(dtype, io, HD, window, normalize):
    tables = rope(HD, 256, "cuda")
    page = 16 if HD != 32 else 7
    pool = Pool(len(LENGTHS), 2, HD, page, -(-201 // page), dtype)
    hist = fill(pool, LENGTHS, 2, HD, io, tables, HD)
    q, k, v = (torch.randn(len(LENGTHS), 2, HD, device="cuda").to(io) for _ in range(3))
    check_decode(pool, LENGTHS, hist, q, window=window, normalize=normalize, tables=tables,
                 tau_window=24, new=(k, v))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F8, I8])
@pytest.mark.parametrize("H,Hk", [(3, 3), (4, 2), (6, 2), (8, 1), (16, 2), (9, 1), (20, 1), (48, 3)])
def test_decode_shared_heads(dtype, H, Hk):
    io = dtype if dtype in ULP else BF16
    lengths = [70, 3, 0, 33]
    pool = Pool(4, Hk, 64, 16, 5, dtype)
    hist = fill(pool, [n + 1 for n in lengths], Hk, 64, io, None, H)
    q = torch.randn(4, H, 64, device="cuda").to(io)
    check_decode(pool, lengths, hist, q, window=None, tau_window=40)
    check_decode(pool, lengths, hist, q, window=33)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
@pytest.mark.parametrize("page,width", [(1, 40), (5, 8), (16, 3), (24, 2), (40, 1), (64, 1)])
def test_decode_rings_of_any_page_size(dtype, page, width):
    """Sequences longer than their table: a ring that has wrapped several times."""
    cap, io = page * width, dtype if dtype in ULP else BF16
    lengths = [cap - 1, cap, cap + 1, 3 * cap + 7, 150]
    tables = rope(64, 400, "cuda")
    pool = Pool(5, 2, 64, page, width, dtype)
    hist = fill(pool, lengths, 2, 64, io, tables, page)
    q, k, v = (torch.randn(5, 2, 64, device="cuda").to(io) for _ in range(3))
    check_decode(pool, lengths, hist, q, window=32, tables=tables, new=(k, v))
    lengths = [t + 1 for t in lengths]
    check_decode(pool, lengths, hist, q, window=None, tau_window=9, tables=tables, new=(v, k))


@gpu
@pytest.mark.parametrize("dtype,HD", [(F32, 64), (BF16, 64), (BF16, 128), (F16, 32), (F8, 64), (I8, 128),
                                      (BF16, 80)])
def test_decode_long_rows_are_split_and_joined(dtype, HD):
    """Few rows and long ones: every length around a piece's ends, in one batch
    with short ones; the same bits on every call."""
    io = dtype if dtype in ULP else BF16
    lengths = [5000, 127, 128, 129, 0, 2047, 2049, -1, 4096]
    pool = Pool(9, 1, HD, 64, 80, dtype)
    hist = fill(pool, [n + 1 for n in lengths], 1, HD, io, None, HD)
    q = torch.randn(9, 2, HD, device="cuda").to(io)
    out, row = check_decode(pool, lengths, hist, q, window=None, tau_window=700)
    for _ in range(5):
        again = paged.paged_tension(q, *pool.cache, int32(lengths), window=None, return_tau=True,
                                    tau_window=700, **pool.scales)
        assert torch.equal(again[0], out) and torch.equal(again[1], row)
    plain = paged.paged_tension(q, *pool.cache, int32(lengths), window=None, **pool.scales)
    assert torch.equal(plain, out)
    check_decode(pool, lengths, hist, q, window=3000, normalize="count")


@gpu
@pytest.mark.parametrize("dtype,H,Hk,HD", [(BF16, 3, 3, 64), (I8, 6, 3, 32), (F16, 24, 3, 64), (F8, 3, 3, 128)])
def test_decode_rows_in_two_pieces(dtype, H, Hk, HD):
    """192 rows of a few hundred keys: two pieces, joined in a cluster, beside
    rows of one piece and of none; new rows written by the piece that ends with them."""
    io = dtype if dtype in ULP else BF16
    lengths = [(37 * i) % 320 for i in range(62)] + [-1, 319]
    tables = rope(HD, 330, "cuda")
    pool = Pool(64, Hk, HD, 16, 20, dtype)
    hist = fill(pool, lengths, Hk, HD, io, tables, HD)
    q = torch.randn(64, H, HD, device="cuda").to(io)
    k, v = (torch.randn(64, Hk, HD, device="cuda").to(io) for _ in "kv")
    check_decode(pool, lengths, hist, q, window=None, tau_window=290, tables=tables, new=(k, v))
    hist = history(pool, [t + 1 if t >= 0 else 0 for t in lengths], Hk, HD)
    check_decode(pool, lengths, hist, q, window=250, normalize="count", tables=tables)


@gpu
@pytest.mark.parametrize("dtype,H,Hk,HD", [(BF16, 2, 2, 64), (F16, 18, 2, 32), (F8, 8, 2, 128), (I8, 2, 2, 64)])
@pytest.mark.parametrize("cap", [496, 1040, 2048])
def test_decode_rows_joined_in_clusters(dtype, H, Hk, HD, cap):
    """Few rows: four to eight pieces in a cluster, rows of fewer pieces, of one
    and of none among them; the longest have wrapped their ring."""
    io = dtype if dtype in ULP else BF16
    lengths = [cap + 5, cap - 1, cap // 2, 130, 129, 1, 0, -1]
    tables = rope(HD, cap + 8, "cuda")
    pool = Pool(8, Hk, HD, 16, cap // 16, dtype)
    hist = fill(pool, lengths, Hk, HD, io, tables, HD)
    q = torch.randn(8, H, HD, device="cuda").to(io)
    k, v = (torch.randn(8, Hk, HD, device="cuda").to(io) for _ in "kv")
    out, row = check_decode(pool, lengths, hist, q, window=None, tau_window=cap, tables=tables, new=(k, v))
    assert ops.last_launches() == 1
    again = paged.paged_tension(q, *pool.cache, int32(lengths), window=None, rope=tables, return_tau=True,
                                tau_window=cap, **pool.scales)
    assert torch.equal(again[0], out) and torch.equal(again[1], row)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F8])
def test_split_step_in_a_graph(dtype):
    """The pieces and the kernel that joins them, captured and replayed with other
    lengths than at the capture."""
    io = dtype if dtype in ULP else BF16
    pool = Pool(2, 1, 64, 16, 200, dtype)
    fill(pool, [3200, 3000], 1, 64, io, None, 4)
    q = torch.randn(2, 1, 64, device="cuda").to(io)
    t = int32([5, 6])
    run = lambda: paged.paged_tension(q, *pool.cache, t, window=None, **pool.scales)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for lens in ([3199, 17], [0, 2999], [130, -1], [1000, 2000]):
        t.copy_(int32(lens))
        q.normal_()
        graph.replay()
        assert torch.equal(out, run())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F8, I8])
@pytest.mark.parametrize("shift", [-60.0, -25.0, 0.0, 40.0])
def test_decode_scores_far_from_zero(dtype, shift):
    """All τ tiny (their mass under the 1e-6 floor, or just their ratio counts),
    or all one: products with τ keep their precision over its whole range."""
    io = dtype if dtype in ULP else F32
    pool = Pool(2, 1, 64, 16, 10, dtype)
    k = torch.randn(2 * 150, 1, 64, device="cuda") * 0.1
    k[..., 0] = shift / 8
    v = torch.randn(2 * 150, 1, 64, device="cuda")
    paged.write_kv(k.to(io), v.to(io), *pool.cache, int32([0, 0]), cu_rows=int32([0, 150, 300]), **pool.scales)
    q = torch.randn(2, 1, 64, device="cuda")
    q[..., 0] = 64.0
    hist = history(pool, [150, 150], 1, 64)
    for normalize in ("mass", "count"):
        for window in (None, 140) if normalize == "mass" else (140,):
            out, _ = check_decode(pool, [149, 149], hist, q.to(io), window=window, normalize=normalize,
                                  tau=False)
            if shift in (-25.0, -60.0) and window:
                # relative: the float64 result over the same keys, scaled up
                ref, _ = orc.decode(q.to(io).cpu().double(), hist, [149, 149], window=window, capacity=160,
                                    scale=8.0, normalize=normalize, tau_width=0)
                # Σ τ·v of 140 terms of both signs: fp32 rounding of each score (|score| ≤ 80,
                # relative error of τ ≤ 80·2^-23·4) against the sum of magnitudes
                size = float(ref.abs().max())
                unit = {F32: 0.0, BF16: 2.0 ** -8, F16: 0.0}[io]
                floor = 2.0 ** -24 if io == F16 else 0.0
                assert float((out.cpu().double() - ref).abs().max()) <= (4e-4 + unit) * size + floor


@gpu
def test_decode_ignores_what_is_out_of_reach():
    """NaN and infinities in rows before the window, after the position, in other
    sequences and in unused pages change nothing."""
    for dtype in (F32, BF16, F16, F8, I8):
        pool = Pool(2, 2, 64, 16, 8, dtype)
        io = dtype if dtype in ULP else BF16
        k, v = (torch.randn(240, 2, 64, device="cuda").to(io) for _ in "kv")
        paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=int32([0, 120, 240]), **pool.scales)
        q = torch.randn(2, 2, 64, device="cuda").to(io)
        hist = history(pool, [120, 120], 2, 64)
        for bad in (math.nan, math.inf, -math.inf):
            x = torch.full((1, 2, 64), bad, device="cuda", dtype=io)
            for pos in list(range(0, 37)) + list(range(70, 128)):  # around 37 … 69
                for b in range(2):
                    one = (pool.k, pool.v, pool.table[b:b + 1])
                    paged.write_kv(x, x, *one, int32([pos]), **pool.scales)
            check_decode(pool, [70, 70], hist, q, window=33)
            check_decode(pool, [69, 69], [(a[:70], b[:70]) for a, b in hist], q, window=32)


@gpu
def test_decode_non_finite_rows_in_reach_poison_their_sequence_only():
    pool = Pool(3, 1, 64, 16, 2, BF16)
    hist = fill(pool, [20, 20, 20], 1, 64, BF16, None, 1)
    x = torch.full((1, 1, 64), math.nan, device="cuda", dtype=BF16)
    paged.write_kv(x, x, pool.k, pool.v, pool.table[1:2], int32([7]))
    q = torch.randn(3, 1, 64, device="cuda", dtype=BF16)
    out = paged.paged_tension(q, *pool.cache, int32([19] * 3), window=None)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()


@gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: rows at its far end."""
    HD, page, Hk = 128, 64, 16
    P = (1 << 32) // (HD * page * Hk) + 9
    try:
        kp, vp = (torch.empty(P, Hk, page, HD, device="cuda", dtype=I8) for _ in "kv")
        ks, vs = (torch.empty(P, Hk, page, device="cuda") for _ in "kv")
    except torch.cuda.OutOfMemoryError:
        pytest.skip("needs 10 GB of free device memory")
    pool = Pool(2, Hk, HD, page, 3, I8)
    far = torch.tensor([[P - 1, 0, P - 5], [P - 2, P - 3, 1]], dtype=torch.int32, device="cuda")
    sc = {"k_scale": ks, "v_scale": vs}
    k, v = (torch.randn(330, Hk, HD, device="cuda", dtype=BF16) for _ in "kv")
    cu, lens = int32([0, 180, 330]), [179, 149]
    tables = rope(HD, 256, "cuda")
    paged.write_kv(k, v, kp, vp, far, int32([0, 0]), cu_rows=cu, rope=tables, **sc)
    paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=cu, rope=tables, **pool.scales)
    q = torch.randn(2, 2 * Hk, HD, device="cuda", dtype=BF16)
    a = paged.paged_tension(q, kp, vp, far, int32(lens), window=None, rope=tables, **sc)
    b = paged.paged_tension(q, *pool.cache, int32(lens), window=None, rope=tables, **pool.scales)
    assert torch.equal(a, b)
    for x, y in zip(paged.read_kv(kp, vp, far, int32([0, 0]), cu, 330, **sc),
                    paged.read_kv(*pool.cache, int32([0, 0]), cu, 330, **pool.scales)):
        assert torch.equal(x, y)


@gpu
def test_strided_queries_and_tables():
    """Views of packed projections, a column slice of a wider page table, and
    queries with a head stride of their own."""
    pool = Pool(3, 2, 64, 16, 4, BF16)
    wide = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:7] = pool.table
    hist = fill(pool, [40, 9, 60], 2, 64, BF16, None, 3)
    pool.table = wide[:, 3:7]
    x = torch.randn(3, 64, 8, device="cuda", dtype=BF16)
    check_decode(pool, [39, 8, 59], hist, x.permute(0, 2, 1)[:, ::2], window=None, tau_window=8)
    y = torch.randn(3, 1 + 6 * 64, device="cuda", dtype=BF16)[:, 1:].unflatten(1, (6, 64))  # rows 2 bytes off
    check_decode(pool, [39, 8, 59], hist, y[:, :4], window=17)


@gpu
def test_other_streams_and_graph_replay():
    """On a side stream behind work there; then a captured step replayed while
    the positions advance on the device."""
    tables = rope(64, 128, "cuda")
    B, H = 4, 3
    lengths = [0, 5, 31, -1]
    seq = [[torch.randn(B, H, 64, device="cuda", dtype=BF16) for _ in range(3)] for _ in range(20)]

    def fresh():
        pool = Pool(B, H, 64, 16, 4, BF16)
        fill(pool, lengths, H, 64, BF16, tables, 5)
        return pool, int32(lengths)

    def one(pool, t, q, k, v):
        a = paged.paged_tension(q, *pool.cache, t, window=24, rope=tables, k=k, v=v)
        b = paged.paged_tension(q, *pool.cache, t, window=None, rope=tables)
        t += (t >= 0).int()
        return a, b

    pool, t = fresh()
    want = [one(pool, t, *x) for x in seq]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    pool, t = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late = [[y * 1 for y in x] for x in seq]  # made on the side stream, after the sleep
        got = [one(pool, t, *x) for x in late]
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    pool, t = fresh()
    buf = [torch.zeros_like(x) for x in seq[0]]
    inactive = torch.full_like(t, -1)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        one(pool, inactive.clone(), *buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(pool, t, *buf)
    for x, w in zip(seq, want):
        for a, b in zip(buf, x):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    ops.poll_device_error("cuda")


# ── refusals ──

@gpu
def test_skipped_indexes_are_reported():
    """Pages outside the pool and positions beyond the RoPE tables: skipped, and
    the device error word says so; the next calls run as before."""
    pool = Pool(2, 1, 64, 16, 4, BF16)
    tables = rope(64, 64, "cuda")
    hist = fill(pool, [40, 40], 1, 64, BF16, tables, 2)
    x = torch.randn(2, 1, 64, device="cuda", dtype=BF16)
    ops.poll_device_error("cuda")
    good = pool.table.clone()

    def reported():
        with pytest.raises(RuntimeError, match="outside"):
            ops.poll_device_error("cuda")
        ops.poll_device_error("cuda")

    for bad in (-1, pool.k.shape[0], 2 ** 31 - 1):
        pool.table[0, 1] = bad
        before = pool.k.clone()
        paged.write_kv(x, x, *pool.cache, int32([20, -1]))
        reported()
        same_bits(pool.k, before, "nothing is written")
        k, v = paged.read_kv(*pool.cache, int32([20, 20]), int32([0, 1, 2]), 2)
        reported()
        assert (k[0] == 0).all() and (v[0] == 0).all() and k[1].abs().max() > 0
        out = paged.paged_tension(x, *pool.cache, int32([39, 39]), window=None, rope=tables)
        reported()
        assert torch.isfinite(out).all()
        pool.table.copy_(good)
    out, tau = paged.paged_tension(x, *pool.cache, int32([64, 39]), window=8, rope=tables, return_tau=True)
    reported()
    assert (out[0] == 0).all() and (tau[0] == 0).all() and tau[1].min() > 0
    paged.write_kv(x, x, *pool.cache, int32([64, -1]), rope=tables)
    reported()
    check_decode(pool, [39, 39], hist, x, window=None, tau_window=4, tables=tables)


@gpu
def test_refusals():
    pool, eight = Pool(2, 2, 64, 16, 4, BF16), Pool(2, 2, 64, 16, 4, F8)
    x, t = torch.randn(2, 2, 64, device="cuda", dtype=BF16), int32([3, 4])
    tables = rope(64, 64, "cuda")

    def no(error, match, fn, *a, **kw):
        with pytest.raises(error, match=match):
            fn(*a, **kw)

    no(ValueError, "scale", paged.write_kv, x, x, *eight.cache, t)
    no(ValueError, "scale", paged.write_kv, x, x, *pool.cache, t, **eight.scales)
    no(ValueError, "one type", paged.write_kv, x, x, pool.k, eight.v, pool.table, t)
    no(ValueError, "contiguous", paged.write_kv, x, x, pool.k.transpose(1, 2), pool.v.transpose(1, 2), pool.table, t)
    no(ValueError, "page_table", paged.write_kv, x, x, pool.k, pool.v, pool.table.long(), t)
    no(ValueError, "page_table", paged.write_kv, x, x, pool.k, pool.v, pool.table.t().contiguous().t(), t)
    no(ValueError, "lengths", paged.write_kv, x, x, *pool.cache, t.long())
    no(ValueError, "lengths", paged.write_kv, x, x, *pool.cache, int32([1, 2, 3]))
    no(ValueError, "one row a sequence", paged.write_kv, x[:1], x[:1], *pool.cache, t)
    no(ValueError, "cu_rows", paged.write_kv, x, x, *pool.cache, t, cu_rows=int32([0, 2]))
    no(ValueError, "v must be", paged.write_kv, x, x[:, :1], *pool.cache, t)
    no(ValueError, "k must be", paged.write_kv, x[..., :32], x, *pool.cache, t)
    no(TypeError, "dtype", paged.write_kv, x.double(), x, *pool.cache, t)
    no(ValueError, "rope", paged.write_kv, x, x, *pool.cache, t, rope=rope(32, 64, "cuda"))
    no(ValueError, "rope", paged.write_kv, x, x, *pool.cache, t, rope=tuple(y.cpu() for y in tables))
    no(RuntimeError, "no gradient", paged.write_kv, x.clone().requires_grad_(), x, *pool.cache, t)
    no(ValueError, "rows", paged.read_kv, *pool.cache, t, int32([0, 1, 2]), -1)
    no(TypeError, "dtype", paged.read_kv, *pool.cache, t, None, 2, dtype=torch.float64)
    no(ValueError, "multiple", paged.paged_tension, x[:, :1], *pool.cache, t, window=8)
    no(ValueError, "W \\+ 1", paged.paged_tension, x, *pool.cache, t, window=64)
    no(ValueError, "window", paged.paged_tension, x, *pool.cache, t, window=0)
    no(ValueError, "count", paged.paged_tension, x, *pool.cache, t, window=None, normalize="count")
    no(ValueError, "normalize", paged.paged_tension, x, *pool.cache, t, window=8, normalize="sum")
    no(ValueError, "tau_window", paged.paged_tension, x, *pool.cache, t, window=None, return_tau=True)
    no(ValueError, "together", paged.paged_tension, x, *pool.cache, t, window=8, k=x)
    no(RuntimeError, "no gradient", paged.paged_tension, x.clone().requires_grad_(), *pool.cache, t, window=8)
    no(RuntimeError, "bad shape", paged.paged_tension, x, *pool.cache, t, window=8, scale=0.0)
    big = Pool(1, 1, 160, 4, 2, BF16)
    y = torch.randn(1, 1, 160, device="cuda", dtype=BF16)
    no(RuntimeError, "unsupported", paged.paged_tension, y, *big.cache, int32([0]), window=None)
    with torch.no_grad():
        paged.write_kv(x.clone().requires_grad_(), x, *pool.cache, t, rope=tables)
    empty = paged.read_kv(*pool.cache, t, int32([0, 0, 0]), 0)
    assert empty[0].shape == (0, 2, 64)


def test_refuses_cpu_tensors():
    pool = Pool(1, 1, 64, 16, 2, BF16, device="cpu")
    x, t = torch.randn(1, 1, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA only"):
        paged.write_kv(x, x, *pool.cache, t)
    with pytest.raises(RuntimeError, match="CUDA only"):
        paged.read_kv(*pool.cache, t, None, 1)
    with pytest.raises(RuntimeError, match="CUDA only"):
        paged.paged_tension(x, *pool.cache, t, window=8)


# ── the C ABI's own checks (no GPU: nothing is launched) ──

def _args(cls):
    a = cls()
    c = a.cache
    c.k_pages = c.v_pages = 1 << 20
    c.dtype, c.pages, c.kv_heads, c.page_size, c.HD, c.batch, c.width = _capi.DT_BF16, 8, 2, 16, 64, 2, 4
    c.table = c.lengths = 1 << 20
    c.table_stride = 4
    return a


@pytest.mark.parametrize("field,value,status", [
    ("pages", 0, 1), ("kv_heads", -1, 1), ("page_size", 0, 1), ("HD", 0, 1), ("batch", 0, 1),
    ("width", 0, 1), ("table_stride", -1, 1), ("dtype", 5, 2), ("dtype", -1, 2), ("HD", 129, 3),
    ("k_pages", None, 5), ("v_pages", None, 5), ("table", None, 5), ("lengths", None, 5),
    ("k_pages", (1 << 20) + 8, 4), ("dtype", _capi.DT_I8, 5), ("k_scale", 1 << 20, 1),
    ("pages", 1 << 30, 3), ("width", 1 << 30, 3)])
def test_abi_refuses_bad_caches(field, value, status):
    lib = _capi.lib()
    calls = ((lib.bozo_paged_write, _args(_capi.PagedWriteArgs)),
             (lib.bozo_paged_read, _args(_capi.PagedReadArgs)),
             (lib.bozo_paged_decode, _args(_capi.PagedDecodeArgs)))
    for fn, a in calls:
        setattr(a.cache, field, value)
        assert fn(a, None) == status
        assert fn(None, None) == 5


def test_abi_refuses_bad_steps():
    lib = _capi.lib()
    w = _args(_capi.PagedWriteArgs)
    w.rows = 3                                  # without cu_rows: one row a sequence
    assert lib.bozo_paged_write(w, None) == 1
    w.rows = 2
    assert lib.bozo_paged_write(w, None) == 5   # no k, v
    w.rope_len = 4
    assert lib.bozo_paged_write(w, None) == 5   # no tables
    r = _args(_capi.PagedReadArgs)
    r.rows = 2
    assert lib.bozo_paged_read(r, None) == 5    # no outputs
    r.out_dtype = _capi.DT_I8
    assert lib.bozo_paged_read(r, None) == 2
    d = _args(_capi.PagedDecodeArgs)
    good = dict(H=4, mode=0, window=8, normalize=1, scale=8.0)

    def status(**over):
        for f, v in dict(good, **over).items():
            setattr(d, f, v)
        return lib.bozo_paged_decode(d, None)

    for over, want in ((dict(H=3), 1), (dict(H=0), 1), (dict(mode=2), 1), (dict(window=0), 1),
                       (dict(window=64), 1), (dict(normalize=3), 1), (dict(scale=0.0), 1), ({}, 5)):
        assert status(**over) == want, over
    d.q.ptr = 1 << 20
    d.q.dtype = _capi.DT_F8E4M3
    assert status() == 2
    d.q.dtype = _capi.DT_BF16
    d.k.ptr = 1 << 20
    assert status() == 5                        # k without v
    d.k.ptr = None
    assert status() == 5                        # no out
    d.out = 1 << 20
    d.out_dtype = _capi.DT_I8
    assert status() == 2
    d.out_dtype, d.tau, d.tau_width = _capi.DT_BF16, 1 << 20, 7
    assert status() == 1                        # a local τ row is the window's
    assert _capi.lib().bozo_paged_decode_workspace(None) == 0


def test_struct_layout_matches_header(tmp_path):
    import ctypes as C
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"bozo_paged_cache": _capi.PagedCache, "bozo_paged_write_args": _capi.PagedWriteArgs,
               "bozo_paged_read_args": _capi.PagedReadArgs, "bozo_paged_decode_args": _capi.PagedDecodeArgs}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"bozo_tension.h\"\n"
                   "int main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    exe = str(tmp_path / "probe")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        key, val = line.split()
        name, _, f = key.partition(".")
        got = getattr(structs[name], f).offset if f else C.sizeof(structs[name])
        assert got == int(val), key
