"""4-bit paged caches (``torch.float4_e2m1fn_x2`` pages of ``bozo_b200.paged``).

* Writing equals the plain fp32 definition bit for bit (codes, group scales, scales).
* Reading equals (code · group) · scale, rounded once to the result's type, bit for bit.
* The decode step is compared with a float64 restatement over the rows as they are
  held, with the bound of the other pages' tests: its operands are exact (e2m1 · e4m3
  has 6 significant bits) but for the query's and τ's second halves (2^-22), its sums
  fp32, its result rounded once: |err| ≤ u·|ref| + 1e-5·max|v|.
* Pools start out full of NaN, so a row read out of reach shows.
"""
import math

import pytest
import torch

from bozo_b200 import _capi, ops, paged
from oracle import paged_oracle as orc
from test_paged import (BF16, F16, F32, Pool, check_decode, fill, history, int32, offsets, rope, same_bits)

F4, F8 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


class Pool4(Pool):
    def __init__(self, B, Hk, HD, page, width, spare=2, device="cuda", allocate=None):
        P = B * width + spare
        order = torch.randperm(P, generator=torch.Generator().manual_seed(P)).int()
        self.table = order[:B * width].view(B, width).clone().to(device)
        for b, n in enumerate(allocate or ()):
            self.table[b, n:] = -1
        shape = (P, Hk, page)
        self.k, self.v = (torch.full((*shape, HD // 2), 0x5a, dtype=torch.uint8, device=device).view(F4) for _ in "kv")
        self.kg, self.vg = (torch.full((*shape, HD // 16), 0x38, dtype=torch.uint8, device=device).view(F8)
                            for _ in "kv")
        self.ks, self.vs = (torch.full(shape, math.nan, device=device) for _ in "kv")
        self.page, self.width, self.cap, self.dtype = page, width, page * width, F4

    @property
    def scales(self):
        return {"k_scale": self.ks, "v_scale": self.vs, "k_group": self.kg, "v_group": self.vg}

    def held(self):
        return [x.view(torch.uint8) for x in (self.k, self.v, self.kg, self.vg)] + [self.ks, self.vs]


def check_write(pool, k, v, start, counts, tables, cu=True):
    want = [x.cpu().clone() for x in pool.held()]
    pos = torch.cat([torch.arange(n) + max(s, 0) for s, n in zip(start, counts)] + [torch.zeros(0, dtype=torch.long)])
    kk, vv = k.cpu().float()[:len(pos)], v.cpu().float()[:len(pos)]
    if tables is not None:
        kk = orc.rotate(kk, tables[0].cpu(), tables[1].cpu(), pos)
    new = [y for pair in zip(orc.hold4(kk), orc.hold4(vv)) for y in pair]  # codes, groups, scales of k and v
    row = 0
    for b, (s, n) in enumerate(zip(start, counts)):
        for i in range(n):
            if s >= 0 and i >= n - pool.cap:
                pid, slot = orc.place(pool.table.cpu(), b, s + i, pool.page)
                for x, y in zip(want, new):
                    x[pid, :, slot] = (y.view(torch.uint8) if y.dtype == F8 else y)[row]
            row += 1
    paged.write_kv(k, v, *pool.cache, int32(start), cu_rows=int32(offsets(counts)) if cu else None,
                   rope=tables, **pool.scales)
    for got, ref, name in zip(pool.held(), want, ("k", "v", "k_group", "v_group", "k_scale", "v_scale")):
        same_bits(got, ref, name)


# ── writing and reading ──

@gpu
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 7), (128, 8), (48, 1), (16, 5), (112, 3), (64, 1)])
def test_write_prompts_bit_for_bit(io, HD, page):
    counts, start = [19, 0, 1, 40, 7], [0, 3, 11, 5, 2]
    pool = Pool4(5, 3, HD, page, -(-48 // page))
    g = torch.Generator("cuda").manual_seed(HD)
    x = torch.randn(sum(counts) + 3, 3 * 3 * HD, generator=g, device="cuda").to(io)  # 3 rows of padding
    _, k, v = (y.unflatten(1, (3, HD)) for y in x.chunk(3, dim=1))
    check_write(pool, k, v, start, counts, rope(HD, 64, "cuda"))


@gpu
def test_write_one_row_a_sequence_skips_inactive_ones():
    pool = Pool4(6, 4, 64, 16, 2)
    k, v = (torch.randn(6, 4, 64, device="cuda", dtype=BF16) for _ in "kv")
    check_write(pool, k, v, [0, -1, 15, 16, 31, 100], [1] * 6, rope(64, 128, "cuda"), cu=False)


@gpu
@pytest.mark.parametrize("HD", [64, 80])
def test_write_longer_than_the_ring_keeps_its_end(HD):
    pool = Pool4(2, 2, HD, 8, 3)
    k, v = (torch.randn(130, 2, HD, device="cuda") for _ in "kv")
    check_write(pool, k, v, [5, 0], [100, 30], rope(HD, 128, "cuda"))


@gpu
def test_write_strided_inputs_and_no_rope():
    k = torch.randn(4, 23, 128, device="cuda")[:, :, ::2].transpose(0, 1)
    v = torch.randn(64, 23, 4, device="cuda", dtype=F16).permute(1, 2, 0)
    check_write(Pool4(1, 4, 64, 16, 2), k, v, [2], [23], None)


@gpu
@pytest.mark.parametrize("HD", [64, 48, 32, 128])
def test_write_rows_that_are_hard_to_quantise(HD):
    """Zeros, halfway codes and halfway group scales, groups far below the row's largest,
    the flush limit and its neighbours, the largest and denormal numbers, infinities
    and NaN."""
    big = torch.finfo(F32).max
    rows = torch.zeros(20, 1, HD)
    rows[1, 0, 3] = -7.5
    level = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i, g in enumerate((448.0, 9.0, 13.0, 0.017578125)):   # halfway between two codes at these group scales
        rows[2 + i] = (level * g).repeat(HD // 8) * torch.where(torch.arange(HD) % 3 == 0, -1.0, 1.0)
        rows[2 + i, 0, HD - 1] = 6 * 448
        rows[2 + i, 0, HD - 2] = torch.nextafter(torch.tensor(2.5 * 448), torch.tensor(0.0))
    for i in range(HD // 16):                                   # group maxima halfway between two e4m3
        rows[6, 0, 16 * i] = 6 * (8.5 + i) * 2.0 ** (i - 3)
        rows[6, 0, 16 * i + 1] = 1.0
    rows[6, 0, HD - 1] = 2688.0
    rows[7] = torch.randn(1, HD) * 2.0 ** -30                   # sixteen that vanish beside the largest
    rows[7, 0, 0] = 1.0
    rows[8, 0, 5], rows[9, 0, 5] = 2.0 ** -80, 2.0 ** -80 * (1 - 2.0 ** -24)
    rows[8, 0, 6], rows[9, 0, 7] = -(2.0 ** -81.3), -(2.0 ** -90)
    rows[10, 0, :] = 1e-41
    rows[11] = (torch.rand(1, HD) * 2 - 1) * 3e38
    rows[12, 0, 1], rows[12, 0, 2], rows[12, 0, 3] = big, 1e-30, -big / 2
    rows[13, 0, 1] = 1.3125 * 2.0 ** 127                        # the last with the smaller scale
    rows[13, 0, 2] = -(2.0 ** 127)
    rows[14, 0, 9] = math.inf
    rows[15, 0, 9], rows[15, 0, 10] = -math.inf, -1.0
    rows[16, 0, 0], rows[16, 0, HD - 1] = math.nan, math.inf
    rows[17, 0, ::2] = -0.0
    rows[18] = torch.randn(1, HD)
    rows[19, 0, :] = 1.3125 * 2.0 ** 11
    pool = Pool4(1, 1, HD, 20, 1)
    check_write(pool, rows.cuda(), rows.flip(0).cuda(), [0], [20], None)
    k, v = paged.read_kv(*pool.cache, int32([0]), int32([0, 20]), 20, dtype=F32, **pool.scales)
    assert torch.isnan(k[14:17]).all() and torch.isnan(v.flip(0)[14:17]).all()
    keep = [i for i in range(20) if not 14 <= i < 17]
    assert torch.isfinite(k[keep]).all() and torch.isfinite(v.flip(0)[keep]).all()
    assert (k[[0, 9, 10, 17]] == 0).all()
    # the definition's error: half a step of e2m1 at the top (1 of 6) and the group scale's
    # half step (2^-4): at most a sixth of the sixteen's largest and a little over
    x, y = rows[keep].double().unflatten(-1, (-1, 16)), k[keep].cpu().double().unflatten(-1, (-1, 16))
    a = x.abs().amax(-1, keepdim=True)
    row = rows[keep].double().abs().amax(-1)[..., None, None]
    ok = (x - y).abs() <= a * (1 + 2.0 ** -4) / 6 + row * 2.0 ** -17 + 2.0 ** -80
    assert bool(ok[[i for i, r in enumerate(keep) if r not in (11, 12, 13)]].all())


@gpu
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 3), (128, 8), (80, 5)])
def test_read_bit_for_bit(out, HD, page):
    counts, start = [33, 0, 5, 17], [4, 0, 9, -1]
    pool = Pool4(4, 3, HD, page, -(-64 // page))
    for x in (pool.k, pool.v):
        x.view(torch.uint8).random_(0, 256)
    for x in (pool.kg, pool.vg):
        x.view(torch.uint8).random_(0, 0x7f)
    for x in (pool.ks, pool.vs):
        x.copy_(torch.exp2(torch.randint(-20, 4, x.shape, device="cuda").float()))
    cu, N = offsets(counts), sum(counts) + 2
    k, v = paged.read_kv(*pool.cache, int32(start), int32(cu), N, dtype=out, **pool.scales)
    for got, (x, g, s) in ((k, (pool.k, pool.kg, pool.ks)), (v, (pool.v, pool.vg, pool.vs))):
        val = orc.unhold4(x.view(torch.uint8).cpu(), g.cpu(), s.cpu())
        ref = torch.zeros(N, 3, HD)
        for b, n in enumerate(counts):
            for i in range(n if start[b] >= 0 else 0):
                pid, slot = orc.place(pool.table.cpu(), b, start[b] + i, page)
                ref[cu[b] + i] = val[pid, :, slot]
        same_bits(got, ref.to(out), "rows")


# ── the decode step ──

LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, -1, 200]


@gpu
@pytest.mark.parametrize("io", [F32, BF16, F16])
@pytest.mark.parametrize("HD,page", [(32, 16), (32, 7), (64, 16), (64, 8), (128, 16), (128, 5), (48, 16), (16, 8)])
@pytest.mark.parametrize("window,normalize", [(16, "mass"), (64, "count"), (1, "none"), (190, "mass"), (None, "mass")])
def test_decode_matches_float64(io, HD, page, window, normalize):
    tables = rope(HD, 256, "cuda")
    pool = Pool4(len(LENGTHS), 2, HD, page, -(-201 // page))
    hist = fill(pool, LENGTHS, 2, HD, io, tables, HD)
    q, k, v = (torch.randn(len(LENGTHS), 2, HD, device="cuda").to(io) for _ in range(3))
    check_decode(pool, LENGTHS, hist, q, window=window, normalize=normalize, tables=tables,
                 tau_window=24, new=(k, v))


@gpu
@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("H,Hk", [(3, 3), (4, 2), (6, 2), (8, 1), (16, 2), (9, 1), (20, 1)])
def test_decode_shared_heads(H, Hk, HD):
    lengths = [70, 3, 0, 33]
    pool = Pool4(4, Hk, HD, 16, 5)
    hist = fill(pool, [n + 1 for n in lengths], Hk, HD, BF16, None, H)
    q = torch.randn(4, H, HD, device="cuda", dtype=BF16)
    check_decode(pool, lengths, hist, q, window=None, tau_window=40)
    check_decode(pool, lengths, hist, q, window=33)


@gpu
@pytest.mark.parametrize("HD", [32, 64])
@pytest.mark.parametrize("page,width", [(1, 40), (5, 8), (16, 3), (24, 2), (40, 1), (64, 1)])
def test_decode_rings_of_any_page_size(HD, page, width):
    cap = page * width
    lengths = [cap - 1, cap, cap + 1, 3 * cap + 7, 150]
    tables = rope(HD, 400, "cuda")
    pool = Pool4(5, 2, HD, page, width)
    hist = fill(pool, lengths, 2, HD, BF16, tables, page)
    q, k, v = (torch.randn(5, 2, HD, device="cuda", dtype=BF16) for _ in range(3))
    check_decode(pool, lengths, hist, q, window=32, tables=tables, new=(k, v))
    lengths = [t + 1 for t in lengths]
    check_decode(pool, lengths, hist, q, window=None, tau_window=9, tables=tables, new=(v, k))


@gpu
@pytest.mark.parametrize("HD,page,H", [(64, 64, 2), (128, 16, 1), (32, 16, 2), (64, 8, 4), (96, 16, 1)])
def test_decode_long_rows_are_split_and_joined(HD, page, H):
    lengths = [5000, 127, 128, 129, 0, 2047, 2049, -1, 4096]
    pool = Pool4(9, 1, HD, page, 5120 // page)
    hist = fill(pool, [n + 1 for n in lengths], 1, HD, BF16, None, HD)
    q = torch.randn(9, H, HD, device="cuda", dtype=BF16)
    out, row = check_decode(pool, lengths, hist, q, window=None, tau_window=700)
    for _ in range(5):
        again = paged.paged_tension(q, *pool.cache, int32(lengths), window=None, return_tau=True,
                                    tau_window=700, **pool.scales)
        assert torch.equal(again[0], out) and torch.equal(again[1], row)
    check_decode(pool, lengths, hist, q, window=3000, normalize="count")


@gpu
@pytest.mark.parametrize("H,Hk,HD", [(3, 3, 64), (6, 3, 32), (24, 3, 128)])
def test_decode_rows_in_two_pieces(H, Hk, HD):
    lengths = [(37 * i) % 320 for i in range(62)] + [-1, 319]
    tables = rope(HD, 330, "cuda")
    pool = Pool4(64, Hk, HD, 16, 20)
    hist = fill(pool, lengths, Hk, HD, BF16, tables, HD)
    q = torch.randn(64, H, HD, device="cuda", dtype=BF16)
    k, v = (torch.randn(64, Hk, HD, device="cuda", dtype=BF16) for _ in "kv")
    check_decode(pool, lengths, hist, q, window=None, tau_window=290, tables=tables, new=(k, v))
    hist = history(pool, [t + 1 if t >= 0 else 0 for t in lengths], Hk, HD)
    check_decode(pool, lengths, hist, q, window=250, normalize="count", tables=tables)


@gpu
@pytest.mark.parametrize("B,H,Hk,HD", [(64, 10, 10, 64), (128, 5, 5, 32), (129, 5, 5, 32), (100, 28, 7, 128)])
def test_decode_many_rows_of_uneven_lengths(B, H, Hk, HD):
    """More blocks than run at a time, sequences of equal lengths and idle ones among them."""
    lengths = [(7 * i * i) % 90 - (i % 11 == 3) * 200 for i in range(B)]
    lengths = [max(t, -1) for t in lengths]
    pool = Pool4(B, Hk, HD, 16, 6)
    hist = fill(pool, [t + 1 for t in lengths], Hk, HD, BF16, None, B)
    q = torch.randn(B, H, HD, device="cuda", dtype=BF16)
    check_decode(pool, lengths, hist, q, window=None, tau_window=50)


@gpu
@pytest.mark.parametrize("shift", [-60.0, -25.0, 0.0, 40.0])
def test_decode_scores_far_from_zero(shift):
    pool = Pool4(2, 1, 64, 16, 10)
    k = torch.randn(2 * 150, 1, 64, device="cuda") * 0.1
    k[..., 0] = shift / 8
    v = torch.randn(2 * 150, 1, 64, device="cuda") * torch.exp2(torch.randint(-30, 30, (300, 1, 1), device="cuda").float())
    paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=int32([0, 150, 300]), **pool.scales)
    q = torch.randn(2, 1, 64, device="cuda")
    q[..., 0] = 64.0
    hist = history(pool, [150, 150], 1, 64)
    check_decode(pool, [149, 149], hist, q, window=None, tau=False)
    check_decode(pool, [149, 149], hist, q, window=140, normalize="count", tau=False)


@gpu
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 16), (128, 8), (80, 16)])
def test_decode_ignores_what_is_out_of_reach(HD, page):
    """NaN rows before the window, after the position, in other sequences, and garbage
    (NaN group scales, NaN and infinite scales) in unused pages change nothing."""
    pool = Pool4(2, 2, HD, page, 128 // page)
    k, v = (torch.randn(240, 2, HD, device="cuda", dtype=BF16) for _ in "kv")
    paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=int32([0, 120, 240]), **pool.scales)
    q = torch.randn(2, 2, HD, device="cuda", dtype=BF16)
    hist = history(pool, [120, 120], 2, HD)
    for scale in (math.nan, math.inf):
        for pos in list(range(0, 37)) + list(range(70, 128)):  # around 37 … 69
            for b in range(2):
                pid, slot = orc.place(pool.table.cpu(), b, pos, page)
                for x in (pool.kg, pool.vg):
                    x.view(torch.uint8)[pid, :, slot] = 0x7f   # a NaN
                pool.ks[pid, :, slot] = pool.vs[pid, :, slot] = scale
        check_decode(pool, [70, 70], hist, q, window=33)
        check_decode(pool, [69, 69], [(a[:70], b[:70]) for a, b in hist], q, window=32)


@gpu
def test_decode_non_finite_rows_in_reach_poison_their_sequence_only():
    for HD in (64, 48):
        pool = Pool4(3, 1, HD, 16, 2)
        fill(pool, [20, 20, 20], 1, HD, BF16, None, 1)
        x = torch.full((1, 1, HD), math.nan, device="cuda", dtype=BF16)
        paged.write_kv(x, x, pool.k, pool.v, pool.table[1:2], int32([7]), **pool.scales)
        q = torch.randn(3, 1, HD, device="cuda", dtype=BF16)
        out = paged.paged_tension(q, *pool.cache, int32([19] * 3), window=None, **pool.scales)
        assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()


@gpu
def test_pages_that_are_not_there():
    """A hole in the table inside the reach: skipped, its τ zero, and reported."""
    pool = Pool4(2, 2, 64, 16, 4)
    hist = fill(pool, [60, 60], 2, 64, BF16, None, 7)
    ops.poll_device_error("cuda")
    pool.table[0, 1] = -1
    q = torch.randn(2, 4, 64, device="cuda", dtype=BF16)
    out, tau = paged.paged_tension(q, *pool.cache, int32([59, 59]), window=None, return_tau=True, tau_window=60,
                                   **pool.scales)
    with pytest.raises(RuntimeError, match="outside"):
        ops.poll_device_error("cuda")
    assert (tau[0, :, 60 - 32:60 - 16] == 0).all() and (tau[0, :, :60 - 32] > 0).all()
    kept = [torch.cat([x[:16], x[32:]]) for x in hist[0]]
    ref, _ = orc.decode(q.cpu().double()[:1], [kept], [43], window=None, capacity=64, scale=8.0, normalize="mass",
                        tau_width=0)
    assert float((out[0].cpu().double() - ref[0]).abs().max()) <= 2.0 ** -7 * float(ref.abs().max()) + 1e-4
    assert torch.isfinite(out).all()


@gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes of codes: rows at its far end."""
    HD, page, Hk = 128, 64, 16
    P = (1 << 32) // (HD // 2 * page * Hk) + 9
    try:
        kp, vp = (torch.empty(P, Hk, page, HD // 2, device="cuda", dtype=torch.uint8).view(F4) for _ in "kv")
        kg, vg = (torch.empty(P, Hk, page, HD // 16, device="cuda", dtype=torch.uint8).view(F8) for _ in "kv")
        ks, vs = (torch.empty(P, Hk, page, device="cuda") for _ in "kv")
    except torch.cuda.OutOfMemoryError:
        pytest.skip("needs 10 GB of free device memory")
    pool = Pool4(2, Hk, HD, page, 3)
    far = torch.tensor([[P - 1, 0, P - 5], [P - 2, P - 3, 1]], dtype=torch.int32, device="cuda")
    sc = {"k_scale": ks, "v_scale": vs, "k_group": kg, "v_group": vg}
    k, v = (torch.randn(330, Hk, HD, device="cuda", dtype=BF16) for _ in "kv")
    cu, lens = int32([0, 180, 330]), [179, 149]
    paged.write_kv(k, v, kp, vp, far, int32([0, 0]), cu_rows=cu, **sc)
    paged.write_kv(k, v, *pool.cache, int32([0, 0]), cu_rows=cu, **pool.scales)
    q = torch.randn(2, 2 * Hk, HD, device="cuda", dtype=BF16)
    a = paged.paged_tension(q, kp, vp, far, int32(lens), window=None, **sc)
    b = paged.paged_tension(q, *pool.cache, int32(lens), window=None, **pool.scales)
    assert torch.equal(a, b)
    for x, y in zip(paged.read_kv(kp, vp, far, int32([0, 0]), cu, 330, **sc),
                    paged.read_kv(*pool.cache, int32([0, 0]), cu, 330, **pool.scales)):
        assert torch.equal(x, y)


@gpu
def test_other_streams_and_graph_replay():
    tables = rope(64, 128, "cuda")
    lengths = [0, 5, 31, -1]
    pool = Pool4(4, 3, 64, 16, 8)
    fill(pool, lengths, 3, 64, BF16, tables, 5)
    q, k, v = (torch.randn(4, 3, 64, device="cuda", dtype=BF16) for _ in range(3))
    t = int32(lengths)
    run = lambda at: paged.paged_tension(q, *pool.cache, at, window=None, rope=tables, k=k, v=v, **pool.scales)
    want = run(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = run(t * 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t)
    for lens in ([1, 6, 32, -1], [2, -1, 33, 0]):
        t.copy_(int32(lens))
        q.normal_()
        graph.replay()
        assert torch.equal(out, run(t))
    ops.poll_device_error("cuda")


# ── refusals ──

@gpu
def test_refusals():
    pool, plain = Pool4(2, 2, 64, 16, 4), Pool(2, 2, 64, 16, 4, BF16)
    x, t = torch.randn(2, 2, 64, device="cuda", dtype=BF16), int32([3, 4])

    def no(match, *at, **scales):
        for call in (lambda: paged.write_kv(x, x, *at, t, **scales),
                     lambda: paged.read_kv(*at, t, None, 2, **scales),
                     lambda: paged.paged_tension(x, *at, t, window=8, **scales)):
            with pytest.raises(ValueError, match=match):
                call()

    full = pool.scales
    no("k_scale", *pool.cache)
    no("k_group", *pool.cache, k_scale=pool.ks, v_scale=pool.vs)
    no("k_group", *pool.cache, **dict(full, v_group=None))
    no("k_group", *plain.cache, k_group=pool.kg, v_group=pool.vg)
    no("k_scale", *pool.cache, k_group=pool.kg, v_group=pool.vg)
    no("group scales", *pool.cache, **dict(full, k_group=pool.kg[..., :2]))
    no("group scales", *pool.cache, **dict(full, k_group=pool.kg.view(torch.uint8)))
    no("group scales", *pool.cache, **dict(full, v_group=pool.vg.cpu()))
    no("group scales", *pool.cache, **dict(full, v_group=pool.vg[1:]))
    no("scales", *pool.cache, **dict(full, v_scale=pool.vs.double()))
    odd = Pool4(2, 2, 64, 16, 4)
    odd.k, odd.v = (torch.zeros(10, 2, 16, 20, dtype=torch.uint8, device="cuda").view(F4) for _ in "kv")
    no("multiple of 16", *odd.cache, **full)
    no("one type", pool.k, plain.v, pool.table, **full)
    ops.poll_device_error("cuda")


def test_refuses_cpu_tensors():
    pool = Pool4(1, 1, 64, 16, 2, device="cpu")
    x, t = torch.randn(1, 1, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: paged.write_kv(x, x, *pool.cache, t, **pool.scales),
                 lambda: paged.read_kv(*pool.cache, t, None, 1, **pool.scales),
                 lambda: paged.paged_tension(x, *pool.cache, t, window=8, **pool.scales)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()


@pytest.mark.parametrize("field,value,status", [
    ("HD", 72, 3), ("HD", 144, 3), ("k_scale", None, 5), ("v_scale", None, 5), ("k_group", None, 5),
    ("v_group", None, 5), ("k_group", (1 << 20) + 8, 4), ("v_group", (1 << 20) + 4, 4)])
def test_abi_refuses_bad_caches(field, value, status):
    lib = _capi.lib()
    for fn, cls in ((lib.bozo_paged_write, _capi.PagedWriteArgs), (lib.bozo_paged_read, _capi.PagedReadArgs),
                    (lib.bozo_paged_decode, _capi.PagedDecodeArgs)):
        a = cls()
        c = a.cache
        c.k_pages = c.v_pages = c.k_scale = c.v_scale = a.k_group = a.v_group = 1 << 20
        c.dtype, c.pages, c.kv_heads, c.page_size, c.HD, c.batch, c.width = _capi.DT_F4E2M1, 8, 2, 16, 64, 2, 4
        c.table = c.lengths = 1 << 20
        c.table_stride = 4
        setattr(a if "group" in field else c, field, value)
        assert fn(a, None) == status


def test_oracle_codes_are_the_nearest_levels():
    """The oracle itself: every code is the nearest level of its quotient in float64."""
    x = torch.randn(50, 64)
    codes, group, scale = orc.hold4(x)
    unit = (group.double() * scale.double()[..., None]).repeat_interleave(16, dim=-1)
    lev = torch.tensor(orc.LEVELS, dtype=torch.float64)
    near = lev[((x.double() / unit).abs()[..., None] - lev).abs().argmin(-1)] * unit * torch.sign(x)
    assert torch.allclose(orc.unhold4(codes, group, scale).double(), near, rtol=1e-7, atol=0)
    assert bool((x.abs().amax(-1) <= 2688 * scale).all()) and bool((x.abs().amax(-1) > 1344 * scale).all())
