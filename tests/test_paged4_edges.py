"""4-bit paged caches at the edges of their interface: argument blocks of hosts that know no
group scales."""
import ctypes as C
import subprocess
import sys

from bozo_b200 import _capi

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
