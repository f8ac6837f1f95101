"""Paged caches (``bozo_b200.paged``) where calls go wrong first: precision of
mixed types, pages that are not there, offsets that do not start at zero,
elements that are not finite."""
import math

import pytest
import torch

from bozo_b200 import ops, paged
from oracle import paged_oracle as orc
from test_paged import (BF16, F8, F16, F32, I8, ULP, Pool, check_decode, fill, history, int32, offsets, plain_write,
                        rope, same_bits)

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


# ── precision ──

@gpu
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2), (3, 1), (8, 2), (5, 1), (16, 2), (11, 1)])
@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("window", [64, None])
def test_fp32_queries_over_bf16_pages_keep_fp32(HD, H, Hk, window):
    """A key's or value's bf16 elements are exact in fp32, so an fp32 step over them
    is as near the float64 result as the same step in plain fp32 operations: its
    score is a sum of three times as many terms (each part of q with each element,
    √3 of the rounding) that the matrix instruction may truncate instead of round
    (twice), hence at most 4 times; an exponential and a reciprocal add 2^-22."""
    B, n = 6, 150
    pool = Pool(B, Hk, HD, 16, 10, BF16)
    hist = fill(pool, [n] * B, Hk, HD, BF16, None, HD + H)
    q = torch.randn(B, H, HD, device="cuda") * 4
    lengths = [n - 1 - i for i in range(B)]
    out, tau = paged.paged_tension(q, *pool.cache, int32(lengths), window=window, return_tau=True,
                                   tau_window=window or n)
    ref = orc.decode(q.cpu().double(), hist, lengths, window=window, capacity=pool.cap, scale=math.sqrt(HD),
                     normalize="mass", tau_width=window or n)
    # the same in fp32, key by key
    want = [torch.zeros_like(x, dtype=F32) for x in ref]
    for b, t in enumerate(lengths):
        hi = t if window else t + 1
        lo = max(0, hi - (window or pool.cap))
        k, v = (x[lo:hi].float().repeat_interleave(H // Hk, dim=1) for x in hist[b])
        row = 1 / (1 + torch.exp(-(q[b].cpu() * k).sum(-1) / math.sqrt(HD)))        # [keys, H]
        want[0][b] = (row[..., None] * v).sum(0) / row.sum(0)[:, None]
        want[1][b, :, :hi - lo] = (row if window else row.flip(0)).T
    for got, plain, exact, name in zip((out, tau), want, ref, ("out", "tau")):
        norm = float(exact.norm())
        err, base = (float((x.cpu().double() - exact).norm()) / norm for x in (got, plain))
        assert err <= 4 * base + 2.0 ** -22, f"{name}: {err:.2e}, plain fp32 {base:.2e}"


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F8, I8])
@pytest.mark.parametrize("H", [1, 4, 8])
@pytest.mark.parametrize("shift", [-60.0, -25.0])
def test_tiny_tau_keep_their_precision(dtype, H, shift):
    """Scores s of up to 80 in size, summed and multiplied by 1/scale and log2 e in
    fp32: at most four roundings of 80 at 2^-23, and as large a relative error of
    τ = e^s, however small."""
    n, tol = 150, 80 * 2.0 ** -23 * 4
    pool = Pool(2, 1, 64, 16, 10, dtype)
    k = torch.randn(2 * n, 1, 64, device="cuda") * 0.1
    k[..., 0] = shift / 8
    v = torch.randn(2 * n, 1, 64, device="cuda")
    paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=int32([0, n, 2 * n]), **pool.scales)
    hist = history(pool, [n, n], 1, 64)
    q = torch.randn(2, H, 64, device="cuda")
    q[..., 0] = 64.0
    out, tau = paged.paged_tension(q, *pool.cache, int32([n - 1] * 2), window=140, normalize="count",
                                   return_tau=True, **pool.scales)
    ref = orc.decode(q.cpu().double(), hist, [n - 1] * 2, window=140, capacity=160, scale=8.0, normalize="count",
                     tau_width=140)
    assert float(((tau.cpu().double() - ref[1]).abs() / ref[1].clamp(min=1e-300)).max()) <= tol
    size = (ref[1].sum(-1) / 140 * float(v.abs().max()))[..., None]    # of the sum of magnitudes
    assert float(((out.cpu().double() - ref[0]).abs() / size).max()) <= tol


# ── pages that are not there ──

@gpu
@pytest.mark.parametrize("dtype,HD", [(BF16, 64), (F16, 32), (F8, 128), (I8, 64), (F32, 64), (BF16, 48), (BF16, 21)])
@pytest.mark.parametrize("page", [16, 8, 5])
@pytest.mark.parametrize("window", [30, None])
def test_exported_tau_of_missing_pages_is_zero(dtype, HD, page, window):
    """Keys whose page is outside the pool are left out: their τ is zero, not what
    the allocator's memory held; the others' τ does not change."""
    io = dtype if dtype in ULP else BF16
    for H, lengths, width in ((2, [47, 40, 45], 48 // page + 1), (6, [47, 40, 45], 48 // page + 1),
                              (2, [600], 620 // page + 1)):   # in one piece; shared heads; in several
        pool = Pool(len(lengths), 2, HD, page, width, dtype)
        hist = fill(pool, [t + 1 for t in lengths], 2, HD, io, None, page)
        q = torch.randn(len(lengths), H, HD, device="cuda").to(io)
        tw = window or max(lengths) + 5
        _, whole = check_decode(pool, lengths, hist, q, window=window, tau_window=tw)
        gone = (lengths[0] - 20) // page                    # in reach of the first sequence
        pool.table[0, gone] = -1
        ops.poll_device_error("cuda")
        keep = torch.full((len(lengths), H, tw), math.nan, device="cuda", dtype=io)
        del keep                                            # the next τ row of this size is that memory
        _, tau = paged.paged_tension(q, *pool.cache, int32(lengths), window=window, return_tau=True,
                                     tau_window=tw, **pool.scales)
        with pytest.raises(RuntimeError, match="outside"):
            ops.poll_device_error("cuda")
        want = whole.clone()
        for pos in range(gone * page, (gone + 1) * page):
            back = lengths[0] - pos
            slot = window - back if window else back
            if 0 <= slot < tw:
                want[0, :, slot] = 0
        assert torch.equal(tau, want)


@gpu
@pytest.mark.parametrize("dtype,HD", [(BF16, 64), (BF16, 32), (F8, 64), (I8, 32), (F32, 64)])
@pytest.mark.parametrize("page", [8, 24, 40, 16, 32, 7, 1])
def test_pages_behind_the_window_may_be_gone(dtype, HD, page):
    """A wide table whose pages wholly before the window have been given back: a
    valid call, wherever the window begins, and no error is reported."""
    io, W = dtype if dtype in ULP else BF16, 20
    lengths = [130 + i for i in range(16)] + [3, W, W + 8]
    pool = Pool(len(lengths), 1, HD, page, 160 // page + 1, dtype)
    hist = fill(pool, lengths, 1, HD, io, None, page)
    for b, t in enumerate(lengths):
        pool.table[b, :max(0, t - W) // page] = -1
    q = torch.randn(len(lengths), 1, HD, device="cuda").to(io)
    ops.poll_device_error("cuda")
    check_decode_of(pool, lengths, hist, q, W)
    ops.poll_device_error("cuda")


def check_decode_of(pool, lengths, hist, q, W):
    out, row = paged.paged_tension(q, *pool.cache, int32(lengths), window=W, return_tau=True, **pool.scales)
    ref = orc.decode(q.cpu().double(), hist, lengths, window=W, capacity=pool.cap, scale=math.sqrt(q.shape[-1]),
                     normalize="mass", tau_width=W)
    big = max([1.0] + [float(v.abs().max()) for _, v in hist])
    for got, want, unit in zip((out, row), ref, (big, 1.0)):
        err = (got.cpu().double() - want).abs()
        assert bool((err <= ULP[q.dtype] * want.abs() + 1e-5 * unit).all())


# ── offsets ──

@gpu
@pytest.mark.parametrize("dtype", [BF16, F8, F32])
@pytest.mark.parametrize("HD", [64, 32, 20])
@pytest.mark.parametrize("first", [1, 5, 40, 300])
def test_rows_before_the_first_offset_are_padding(dtype, HD, first):
    """Offsets into a longer packed batch: rows before ``cu_rows[0]`` are padding as
    those from ``cu_rows[B]`` on are, whichever kernel takes the call."""
    counts, start = [9, 0, 1, 30], [0, 3, 11, 5]
    cu = [first + x for x in offsets(counts)]
    rows = cu[-1] + 3
    tables = rope(HD, 64, "cuda")
    pool = Pool(4, 3, HD, 16, 4, dtype)
    k, v = (torch.randn(rows, 3, HD, device="cuda", dtype=BF16) for _ in "kv")
    want = plain_write(pool, k[first:], v[first:], start, counts, tables)
    paged.write_kv(k, v, *pool.cache, int32(start), cu_rows=int32(cu), rope=tables, **pool.scales)
    for got, ref, name in zip((pool.k, pool.v, pool.ks, pool.vs), want, ("k_pages", "v_pages", "k_scale", "v_scale")):
        if got is not None:
            same_bits(got.cpu(), ref, name)
    shifted = paged.read_kv(*pool.cache, int32(start), int32(cu), rows, **pool.scales)
    plain = paged.read_kv(*pool.cache, int32(start), int32(offsets(counts)), rows - first, **pool.scales)
    for x, y in zip(shifted, plain):
        assert (x[:first] == 0).all()
        same_bits(x[first:], y, "read")


# ── elements that are not finite ──

@gpu
@pytest.mark.parametrize("dtype,HD", [(BF16, 64), (F16, 64), (F32, 64), (F8, 64), (I8, 64), (BF16, 48), (F16, 21)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_one_element_that_is_not_finite(dtype, HD, bad, where):
    """In one key, one value or one query: a NaN spoils the outputs that reach it (a
    16- or 32-bit value's only in its own column), and nothing else changes: not
    other sequences, other key heads or, for a query, other heads.  An infinite key
    or query gives τ 0 or 1, or NaN, an infinite value no finite number."""
    io = dtype if dtype in ULP else BF16
    n, H, Hk = 40, 4, 2
    q = torch.randn(3, H, HD, device="cuda").to(io)
    k, v = (torch.randn(3 * n, Hk, HD, device="cuda").to(io) for _ in "kv")
    outs = []
    for spoil in (False, True):
        pool, qq, kk, vv = Pool(3, Hk, HD, 16, 3, dtype), q.clone(), k.clone(), v.clone()
        if spoil:
            if where == "query":
                qq[1, 2, 5] = bad
            else:
                (kk if where == "key" else vv)[n + 17, 1, 5] = bad
        paged.write_kv(kk, vv, *pool.cache, int32([0] * 3), cu_rows=int32([0, n, 2 * n, 3 * n]), **pool.scales)
        outs.append(paged.paged_tension(qq, *pool.cache, int32([n - 1] * 3), window=None, return_tau=True,
                                        tau_window=n, **pool.scales))
    (good, _), (got, tau) = outs
    hit = torch.zeros_like(got, dtype=torch.bool)
    if where == "query":
        hit[1, 2] = True
    elif where == "value" and dtype in ULP:
        hit[1, 2:, 5] = True
    else:
        hit[1, 2:] = True
    assert torch.equal(got[~hit], good[~hit])
    if math.isnan(bad) or (dtype not in ULP and where != "query"):   # an 8-bit row with either is all NaN
        assert torch.isnan(got[hit]).all()
    elif where == "value":
        assert not torch.isfinite(got[hit]).any()
    else:
        tau = tau[1, 2] if where == "query" else tau[1, 2:, n - 1 - 17]
        assert ((tau == 0) | (tau == 1) | torch.isnan(tau)).all()


# ── what a call says of itself ──

@gpu
@pytest.mark.parametrize("dtype,HD,path", [(BF16, 64, "mma"), (F16, 128, "mma"), (F8, 32, "mma"), (I8, 64, "mma"),
                                           (F32, 64, "simt"), (BF16, 48, "simt"), (I8, 21, "simt")])
def test_last_path_names_the_kernel(dtype, HD, path):
    pool = Pool(1, 1, HD, 16, 2, dtype)
    x = torch.randn(1, 1, HD, device="cuda").to(dtype if dtype in ULP else BF16)
    paged.write_kv(x, x, *pool.cache, int32([0]), **pool.scales)
    assert ops.last_path() == "simt"
    paged.paged_tension(x, *pool.cache, int32([0]), window=None, **pool.scales)
    assert ops.last_path() == path and ops.last_launches() == 1


@gpu
def test_misaligned_pages_are_refused_by_name():
    pages = torch.zeros(1 + 2 * 2 * 16 * 64, device="cuda", dtype=BF16)[1:].view(2, 2, 16, 64)
    x, table = torch.randn(1, 2, 64, device="cuda", dtype=BF16), int32([[0]])
    with pytest.raises(RuntimeError, match="aligned pages"):
        paged.write_kv(x, x, pages, pages, table, int32([0]))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("B,launches", [(192, 1), (1024, 2)])
def test_two_pieces_joined_in_a_cluster_or_by_a_kernel(dtype, B, launches):
    """Pieces are joined in clusters where these all find their place at once, else by
    a second kernel: with the same result as a few rows, cut up further, give."""
    n = 640 if B == 192 else 4200
    pool = Pool(1, 1, 32, 16, -(-n // 16), dtype)
    fill(pool, [n], 1, 32, BF16, None, B)
    lengths = [(i * 131) % n for i in range(B)]
    q = torch.randn(B, 1, 32, device="cuda", dtype=BF16)

    def run(rows):
        table = pool.table.expand(len(rows), -1).contiguous()
        return paged.paged_tension(q[rows], pool.k, pool.v, table, int32([lengths[i] for i in rows]), window=None,
                                   **pool.scales).float()

    out = run(list(range(B)))
    assert ops.last_launches() == launches
    some = list(range(0, B, B // 8))
    torch.testing.assert_close(out[some], run(some), rtol=2.0 ** -7, atol=1e-5)


@gpu
@pytest.mark.parametrize("dtype,HD", [(BF16, 64), (F8, 32), (F32, 64), (F16, 48), (I8, 21)])
@pytest.mark.parametrize("page", [16, 8, 3])
def test_positions_up_to_the_largest(dtype, HD, page):
    """The last positions that 32 bits hold give what the same rows give at the start
    of their ring."""
    cap, top = 48, 2 ** 31 - 1
    io = dtype if dtype in ULP else BF16
    for t in (top, top - 1, top - 20):
        low = t % cap + cap                           # the same rows of the ring
        k, v = (torch.randn(cap, 2, HD, device="cuda").to(io) for _ in "kv")
        q, nk, nv = (torch.randn(1, 2, HD, device="cuda").to(io) for _ in range(3))
        got = []
        for at in (t, low):
            pool = Pool(1, 2, HD, page, cap // page, dtype)
            cu = int32([0, cap])
            paged.write_kv(k, v, *pool.cache, int32([at - cap]), cu_rows=cu, **pool.scales)
            got.append([*paged.read_kv(*pool.cache, int32([at - cap]), cu, cap, **pool.scales),
                        *paged.paged_tension(q, *pool.cache, int32([at]), window=30, k=nk, v=nv, return_tau=True,
                                             **pool.scales),
                        *paged.paged_tension(q, *pool.cache, int32([at]), window=None, return_tau=True,
                                             tau_window=cap, **pool.scales), pool.k, pool.v])
        for x, y in zip(*got):
            same_bits(x, y, f"position {t}")
    ops.poll_device_error("cuda")
