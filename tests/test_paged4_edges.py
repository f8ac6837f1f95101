"""4-bit paged caches at their edges: argument blocks of hosts that know no group scales,
rows whose groups are of very different sizes."""
import ctypes as C
import math
import subprocess
import sys

import pytest
import torch

from bozo_b200 import _capi, paged
from oracle import paged_oracle as orc
from test_paged import history, int32, offsets
from test_paged4 import Pool4

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


ENTRY = {"write": ("bozo_paged_write", _capi.PagedWriteArgs), "read": ("bozo_paged_read", _capi.PagedReadArgs),
         "decode": ("bozo_paged_decode", _capi.PagedDecodeArgs),
         "workspace": ("bozo_paged_decode_workspace", _capi.PagedDecodeArgs)}


def block_before_unmapped_memory(cls, size):
    """An argument block of which `size` bytes are there: what follows may not be touched."""
    libc, page = C.CDLL(None, use_errno=True), 65536
    libc.mmap.restype, libc.mmap.argtypes = C.c_void_p, [C.c_void_p, C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_long]
    libc.mprotect.argtypes = [C.c_void_p, C.c_size_t, C.c_int]
    base = libc.mmap(None, 2 * page, 3, 0x22, -1, 0)                # private, anonymous
    assert base not in (None, C.c_void_p(-1).value) and libc.mprotect(base + page, page, 0) == 0
    return cls.from_address(base + page - size)


def call_with_short_block(entry, dtype):
    """The call's status; its pointers are no device's, so nothing is launched on any machine."""
    name, cls = ENTRY[entry]
    a = block_before_unmapped_memory(cls, cls.k_group.offset)
    c, at = a.cache, 1 << 20
    c.k_pages = c.v_pages = c.table = c.lengths = at
    c.dtype, c.pages, c.kv_heads, c.page_size, c.HD, c.batch, c.width, c.table_stride = dtype, 8, 2, 16, 64, 2, 4, 4
    if dtype in (_capi.DT_F8E4M3, _capi.DT_I8):
        c.k_scale = c.v_scale = at
    if cls is _capi.PagedDecodeArgs:
        a.H, a.mode, a.window, a.normalize, a.scale = 2, _capi.MODE_LOCAL, 8, _capi.NORM_MASS, 8.0
        a.q.ptr = a.out = at
    else:
        a.rows = 2
        for f in ("k", "v") if entry == "write" else ():
            getattr(a, f).ptr = at
        if entry == "read":
            a.k_out = a.v_out = at
    return getattr(_capi.lib(), name)(C.byref(a), *(() if entry == "workspace" else (None,)))


OTHERS = (_capi.DT_F32, _capi.DT_BF16, _capi.DT_F16, _capi.DT_F8E4M3, _capi.DT_I8)
BOZO_ERR_CUDA = 7


def test_blocks_of_other_pages_may_end_before_the_group_scales():
    """``k_group`` and ``v_group`` came behind the fields that earlier hosts were built with, and
    are read for 4-bit pages only.  A child makes the calls: reading past a block ends it."""
    code = (f"import sys; sys.path[:0] = {sys.path!r}\nimport test_paged4_edges as t\n"
            "for e in t.ENTRY:\n    print(e, *(t.call_with_short_block(e, d) for d in t.OTHERS), flush=True)")
    child = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    got = dict(line.split(maxsplit=1) for line in child.stdout.splitlines())
    assert child.returncode == 0 and list(got) == list(ENTRY), (child.returncode, got, child.stderr[-2000:])
    # all checks passed, up to the pointers, which are not a device's (the query needs no device)
    for entry in ("write", "read", "decode"):
        assert [int(x) for x in got[entry].split()] == [BOZO_ERR_CUDA] * len(OTHERS), entry


# ── groups of different sizes in one row ──

def sized_rows(rows, Hk, HD, small, mixed, seed):
    """Normal rows whose groups but one are 2^-small of it (`mixed`: that one changes from
    key to key, so every group is large somewhere)."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(rows, Hk, HD // 16, 16, generator=g, device="cuda")
    large = torch.zeros(rows, dtype=torch.long, device="cuda")
    if mixed:
        large = torch.randint(0, HD // 16, (rows,), generator=g, device="cuda")
    size = torch.full((rows, HD // 16), 2.0 ** -small, device="cuda").scatter_(1, large[:, None], 1.0)
    return (x * size[:, None, :, None]).flatten(-2)


@gpu
@pytest.mark.parametrize("small", [4, 8, 11, 14, 17])
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2), (8, 2), (7, 1)])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 16), (128, 16), (64, 8), (128, 5), (32, 5), (48, 16)])
def test_small_groups_keep_their_precision(HD, page, H, Hk, small):
    """|err| ≤ 1e-5 · the column's own largest |v|, whatever the row's other groups hold.

    Queries of a quarter keep Σ|q·k| / √HD under 2, so with mass normalisation the parts are:
    q as two halfs, 2^-23 of each term, and a score's sums, a dozen additions of 2^-23: dz <
    3e-6, which moves τ by (1 − τ)·dz and the quotient by twice that, < 4.5e-6; the sigmoid's
    two approximations, 2^-21, twice: 1e-6; τ (times the row's scale) as two halfs, 2^-21 of
    the largest, which is at most 3 times the mean: 1.5e-6; sums of products, of warps and
    pieces, a dozen additions: 1.5e-6; the result's own 2^-24.  Below 1e-5 together."""
    lengths = [0, 39, 299]
    pool = Pool4(3, Hk, HD, page, -(-300 // page))
    counts = [n + 1 for n in lengths]
    for mixed in (False, True):
        k = sized_rows(sum(counts), Hk, HD, small, mixed, HD + small)
        v = sized_rows(sum(counts), Hk, HD, small, mixed, HD + small + 1)
        paged.write_kv(k, v, *pool.cache, int32([0] * 3), cu_rows=int32(offsets(counts)), **pool.scales)
        hist = history(pool, counts, Hk, HD)
        q = torch.randn(3, H, HD, device="cuda") * 0.25
        for window in (None, 24):
            out = paged.paged_tension(q, *pool.cache, int32(lengths), window=window, **pool.scales)
            ref, _ = orc.decode(q.cpu().double(), hist, lengths, window=window, capacity=pool.cap, scale=math.sqrt(HD),
                                normalize="mass", tau_width=0)
            for b, t in enumerate(lengths):
                lo, end = (0, t + 1) if window is None else (max(0, t - window), t)
                if end == lo:
                    assert (out[b] == 0).all()
                    continue
                top = hist[b][1][lo:end].abs().amax(0).repeat_interleave(H // Hk, dim=0)   # [H, HD]
                err = (out[b].cpu().double() - ref[b]).abs()
                assert bool((err <= 1e-5 * top).all()), (b, float((err / top.clamp(min=1e-30)).max()))
