"""Page tables at their edges: pages that a fork may lack, calls of two threads at once."""
import ctypes as C
import random
import threading

import pytest
import torch

from bozo_b200 import _capi, ops, paged
from oracle import paged_oracle as orc
from test_page_tables import check_fork, int32

gpu = pytest.mark.gpu

# rows of 16 and 17 tokens on pages of 16, the first page shared, both to follow the second
SHARED = ([[0, -1], [0, 1]], [16, 17], [1, 1], [2, 1], 16)


def test_as_many_rows_may_want_a_page_more():
    """The counterexample by hand: the shared page stays, so nothing is given up."""
    table, refs, copies, missing = orc.fork(*SHARED, True)
    assert missing == 1 and refs == [2, 1] and table == [[0, 1], [0, -1]] and copies == [(-1, -1)] * 2


@gpu
def test_fork_reports_the_page_that_sharing_lacks():
    assert check_fork(*SHARED, True)[3] == 1
    table, lengths, parents, refs, page = SHARED
    assert check_fork(table, lengths, parents, refs + [0], page, True)[3] == 0


@gpu
@pytest.mark.parametrize("share", [True, False])
def test_a_page_for_every_entry_is_enough(share):
    """Generations of forks that multiply one row at its fullest, with no spare page."""
    rng = random.Random(7)
    B, M, page = 6, 4, 5
    table, lengths = [[-1] * M for _ in range(B)], [-1] * B
    refs = [0] * (B * M)
    lengths[0] = 0
    for gen in range(40):
        tokens = [rng.randint(0, min(6, M * page - t)) if t >= 0 else 0 for t in lengths]
        table, refs, _, missing, _ = orc.reserve(table, lengths, tokens, refs, page, 0)
        assert missing == 0
        lengths = [t + n if t >= 0 else t for t, n in zip(lengths, tokens)]
        alive = [b for b in range(B) if lengths[b] >= 0]
        parents = [rng.choice(alive[:1 + gen % len(alive)]) for _ in range(B)]
        table, refs, _, missing = check_fork(table, lengths, parents, refs, page, share)
        assert missing == 0
        lengths = [lengths[x] for x in parents]
        if all(t == M * page for t in lengths):                 # full: all but one go, and begin again
            table, refs, _, _ = check_fork(table, lengths, [-1] * B, refs, page, share)
            lengths = [0] + [-1] * (B - 1)
            assert sum(refs) == 0


def idle_call(name, B, M, P=20000, page=4):
    """An argument block over idle rows, and what it points to."""
    int32 = lambda *shape, value=-1: torch.full(shape, value, dtype=torch.int32, device="cuda")
    t = {"table": int32(B, M), "lengths": int32(B), "refs": int32(P, value=0), "missing": int32(1)}
    if name == "fork":
        a = _capi.PagedForkArgs()
        a.share, t["parents"], t["copies"] = 1, int32(B), int32(B, 2)
    else:
        a = _capi.PagedReserveArgs()
        t["cu_rows"] = int32(B + 1)
    a.batch, a.width, a.table_stride, a.page_size, a.pages = B, M, M, page, P
    for field, x in t.items():
        setattr(a, field, x.data_ptr())
    return a, t


@gpu
@pytest.mark.parametrize("name", ["fork", "reserve"])
def test_calls_of_several_sizes_from_two_threads(name):
    """The C entries from two threads (which ctypes lets run), each with tables of its own that
    want different amounts of shared memory: every call is launched."""
    call = getattr(_capi.lib(), f"bozo_paged_{name}")
    blocks = [idle_call(name, 8192, 2), idle_call(name, 1500 if name == "fork" else 4000, 8)]
    status = [set(), set()]

    def run(i):
        stream = torch.cuda.Stream()
        for _ in range(3000):
            status[i].add(call(C.byref(blocks[i][0]), stream.cuda_stream))
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert status == [{0}, {0}]
    for a, t in blocks:
        assert int(t["missing"]) == 0 and (t["table"] == -1).all() and (t["refs"] == 0).all()


@gpu
def test_the_last_pages_that_31_bits_number():
    """A pool of 2^31 − 1 pages, all taken but three of its last: its last word of 32 pages ends
    where an int does."""
    P = 2 ** 31 - 1
    try:
        refs = torch.ones(P, dtype=torch.int32, device="cuda")
    except torch.cuda.OutOfMemoryError:
        pytest.skip("needs 9 GB of free device memory")
    refs[[-40, -7, -1]] = 0
    table = int32([[5, -1, -1], [-1, -1, -1]])
    plan = paged.reserve(table, int32([1, -1]), int32([2, 0]), refs, 1, rows=3)
    assert table.tolist() == [[5, P - 40, P - 7], [-1] * 3] and plan.missing.item() == 0
    assert plan.slot.tolist() == [P - 40, P - 7, -1]
    plan = paged.reserve(table, int32([3, 0]), int32([0, 2]), refs, 1)
    assert plan.missing.item() == 1 and table[1].tolist() == [-1] * 3      # one is left
    copies, missing = paged.fork(table, int32([3, -1]), int32([0, 0]), refs, 1, share=False)
    assert missing.item() == 2 and table.tolist() == [[5, P - 40, P - 7], [P - 1, -1, -1]]
    assert copies.tolist() == [[-1, -1]] * 3 + [[5, P - 1], [-1, -1], [-1, -1]]
    assert refs[-40:].sum().item() == 40


@gpu
@pytest.mark.parametrize("rows", [9, 5000])      # places by the first kernel, and by their own
def test_positions_end_at_31_bits(rows):
    """Tokens behind the last position that an int holds have none (they had negative ones)."""
    last = 2 ** 31 - 1
    table, refs = int32([[3, 1], [0, 2], [-1, -1]]), int32([1, 1, 1, 1])
    ops.poll_device_error("cuda")
    plan = paged.reserve(table, int32([last - 2, last - 1, 0]), int32([3, 2, 0]), refs, 16, rows=rows)
    ops.poll_device_error("cuda")                  # the last position is one
    slots = [1 * 16 + 13, 1 * 16 + 14, 1 * 16 + 15, 2 * 16 + 14, 2 * 16 + 15]   # 2^31 − 1 = 31 mod 32
    assert plan.pos[:5].tolist() == [last - 2, last - 1, last, last - 1, last] and plan.slot[:5].tolist() == slots
    plan = paged.reserve(table, int32([last - 2, last, -1]), int32([5, 1, 3]), refs, 16, rows=rows)
    with pytest.raises(RuntimeError, match="outside"):
        ops.poll_device_error("cuda")
    assert plan.cu_rows.tolist() == [0, 5, 6, 6] and plan.seq[:7].tolist() == [0] * 5 + [1, -1]
    assert plan.pos[:7].tolist() == [last - 2, last - 1, last, -1, -1, last, -1]
    assert plan.slot[:7].tolist() == [29, 30, 31, -1, -1, 47, -1]
    assert (plan.pos[7:] == -1).all() and plan.missing.item() == 0 and table.tolist() == [[3, 1], [0, 2], [-1, -1]]
