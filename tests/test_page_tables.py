"""Page tables on the device (``paged.reserve``, ``paged.fork``, ``paged.copy_pages``)
against lists worked through one entry at a time.  Everything is a whole number: the
results are equal, and entries that a call does not own stay as they were."""
import random

import pytest
import torch

from bozo_b200 import _capi, ops, paged
from oracle import paged_oracle as orc

gpu = pytest.mark.gpu


def int32(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def random_tables(rng, B, M, page, lengths, spare):
    held = [min(M, -(-max(t, 0) // page)) for t in lengths]
    order = list(range(sum(held) + spare))
    rng.shuffle(order)
    table, refs = [[-1] * M for _ in range(B)], [0] * len(order)
    for row, n in zip(table, held):
        for j in range(n):
            row[j] = order.pop()
            refs[row[j]] = 1
    return table, refs


def check_reserve(table, lengths, tokens, refs, page, rows):
    want = orc.reserve(table, lengths, tokens, refs, page, rows)
    wide = torch.full((len(table), len(table[0]) + 3), 77, dtype=torch.int32, device="cuda")
    dev = wide[:, 1:-2]  # rows of a wider table
    dev.copy_(int32(table))
    r = int32(refs)
    plan = paged.reserve(dev, int32(lengths), int32(tokens), r, page, rows=rows)
    assert dev.tolist() == want[0] and r.tolist() == want[1]
    assert plan.cu_rows.tolist() == want[2] and plan.missing.tolist() == [want[3]]
    assert list(zip(plan.seq.tolist(), plan.pos.tolist(), plan.slot.tolist())) == want[4]
    assert (wide[:, 0] == 77).all() and (wide[:, -2:] == 77).all()
    return want


# ── reserve ──

@gpu
@pytest.mark.parametrize("B", [1, 3, 64, 1100])
@pytest.mark.parametrize("page,M", [(16, 12), (1, 40), (7, 9), (64, 2)])
def test_reserve_ragged_tokens(B, page, M):
    rng = random.Random(B * 100 + page)
    cap = M * page
    lengths = [rng.choice([0, 1, page, cap - 1, cap, -1, rng.randint(0, cap)]) for _ in range(B)]
    tokens = [rng.choice([0, 1, 1, page, rng.randint(0, cap), -3]) for _ in range(B)]
    table, refs = random_tables(rng, B, M, page, lengths, spare=B * M + 5)
    n = sum(max(0, x) for x, t in zip(tokens, lengths) if t >= 0)
    check_reserve(table, lengths, tokens, refs, page, n + 4)


@gpu
def test_reserve_rings_and_tokens_past_them():
    """More tokens than the ring holds: the earlier ones have no slot; a table that is
    full gets no page."""
    table, refs = random_tables(random.Random(1), 3, 4, 8, [100, 20, 0], spare=9)
    check_reserve(table, [100, 20, 0], [50, 40, 33], refs, 8, 130)


@gpu
def test_reserve_keeps_what_was_reserved_before():
    rng = random.Random(2)
    table, refs = random_tables(rng, 4, 8, 16, [5, 16, 33, -1], spare=20)
    first = check_reserve(table, [5, 16, 33, -1], [30, 40, 1, 9], refs, 16, 80)
    again = check_reserve(first[0], [5, 16, 33, -1], [30, 40, 1, 9], first[1], 16, 80)
    assert again[0] == first[0] and again[1] == first[1]
    check_reserve(first[0], [5, 16, 33, 0], [60, 41, 70, 20], first[1], 16, 200)


@gpu
@pytest.mark.parametrize("P", [1, 5, 4095, 70001])
def test_reserve_all_or_nothing(P):
    """One page too few: no table row changes, and the count is reported; then just enough,
    the free pages scattered over the pool."""
    rng = random.Random(P)
    B, M, page = 2, max(1, P // 2 + 1), 4
    refs = [rng.choice([0, 0, 1, 3]) for _ in range(P)]
    free = refs.count(0)
    a = min(M, free // 2)
    b = min(M, free - a)
    table = [[-1] * M, [P] * M]   # both are empty entries
    if a + b < 2 * M:
        check_reserve(table, [0, 0], [a * page, min(M, b + 1) * page], refs, page, 3)
    if a + b:
        got = check_reserve(table, [0, 0], [a * page - 3 if a else 0, b * page], refs, page, 7)
        assert got[3] == 0


@gpu
def test_reserve_one_each_and_no_rows():
    table, refs = int32([[3, -1], [-1, -1], [0, 1]]), int32([1, 1, 0, 1, 0])
    plan = paged.reserve(table, int32([16, 0, -1]), None, refs, 16)
    assert table.tolist() == [[3, 2], [4, -1], [0, 1]] and refs.tolist() == [1] * 5
    assert plan.cu_rows.tolist() == [0, 1, 2, 2] and plan.missing.tolist() == [0]
    assert plan.seq is plan.pos is plan.slot is None
    plan = paged.reserve(table, int32([17, 1, -1]), None, refs, 16, rows=0)
    assert plan.seq.shape == (0,)


@gpu
def test_reserve_absurd_counts_are_reported():
    table, refs = int32([[-1, -1], [-1, -1]]), int32([0, 0, 0])
    ops.poll_device_error("cuda")
    plan = paged.reserve(table, int32([0, 0]), int32([2 ** 31 - 1, 5]), refs, 4, rows=6)
    with pytest.raises(RuntimeError, match="outside"):
        ops.poll_device_error("cuda")
    assert plan.cu_rows.tolist() == [0, 0, 5] and table.tolist() == [[-1, -1], [0, 1]]


# ── fork ──

def check_fork(table, lengths, parents, refs, page, share):
    want = orc.fork(table, lengths, parents, refs, page, share)
    dev, r = int32(table), int32(refs)
    copies, missing = paged.fork(dev, int32(lengths), int32(parents), r, page, share=share)
    assert dev.tolist() == want[0] and r.tolist() == want[1]
    assert [tuple(x) for x in copies.tolist()] == want[2] and missing.tolist() == [want[3]]
    return want


@gpu
@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("B,M,page", [(1, 1, 1), (4, 9, 16), (60, 12, 5), (300, 40, 8), (2000, 5, 4), (2300, 5, 4), (5000, 3, 2)])
def test_fork_generations(share, B, M, page):
    """Rows that multiply, go and grow over several steps; pages come back."""
    rng = random.Random(B)
    cap = M * page
    lengths = [rng.choice([-1, 0, 1, page, rng.randint(0, cap)]) for _ in range(B)]
    table, refs = random_tables(rng, B, M, page, lengths, spare=3)
    for gen in range(4):
        alive = [b for b in range(B) if lengths[b] >= 0] or [0]
        few = rng.sample(alive, max(1, len(alive) // 3))
        parents = [rng.choice([rng.choice(few), rng.choice(alive), b if lengths[b] >= 0 else -1]) for b in range(B)]
        if gen == 1:
            parents = [rng.choice([-1, x]) for x in parents]
        table, refs, _, _ = check_fork(table, lengths, parents, refs, page, share)
        lengths = [lengths[x] if x >= 0 else -1 for x in parents]
        held = [sum(p in row for row in table) for p in range(len(refs))] if B <= 300 else refs
        assert held == refs
        want = orc.reserve(table, lengths, [rng.randint(0, max(0, min(3, cap - t))) for t in lengths], refs, page, 0)
        if not want[3]:
            table, refs = want[0], want[1]
            lengths = [t + n if t >= 0 else t for t, n in zip(lengths, [b - a for a, b in zip(want[2], want[2][1:])])]


@gpu
def test_fork_identity_and_release():
    table, refs = random_tables(random.Random(3), 5, 6, 8, [40, 3, 48, 0, -1], spare=4)
    got = check_fork(table, [40, 3, 48, 0, -1], [0, 1, 2, 3, 4], refs, 8, True)
    assert got[0] == table and got[1] == refs
    got = check_fork(table, [40, 3, 48, 0, -1], [-1] * 5, refs, 8, False)
    assert set(got[1]) == {0}


@gpu
@pytest.mark.parametrize("share", [True, False])
def test_fork_too_few_pages(share):
    table, refs = random_tables(random.Random(4), 4, 4, 8, [20, -1, -1, -1], spare=2)
    got = check_fork(table, [20, -1, -1, -1], [0, 0, 0, 0], refs, 8, share)
    assert got[3] == (1 if share else 7)


@gpu
def test_fork_bad_parents_and_rings_that_share_are_reported():
    table, refs = random_tables(random.Random(5), 3, 2, 4, [5, 8, 3], spare=3)
    ops.poll_device_error("cuda")
    check_fork(table, [5, 8, 3], [1, 3, 2 ** 31 - 1], refs, 4, True)   # the last two: emptied
    with pytest.raises(RuntimeError, match="outside"):
        ops.poll_device_error("cuda")
    check_fork(table, [5, 8, 3], [1, 1, 2], refs, 4, True)
    ops.poll_device_error("cuda")
    check_fork(table, [5, 9, 3], [1, 1, 2], refs, 4, True)
    with pytest.raises(RuntimeError, match="outside"):
        ops.poll_device_error("cuda")


# ── copies ──

@gpu
@pytest.mark.parametrize("n_pools", [1, 7, 131, 300])
def test_copy_pages(n_pools):
    """Pools of any type and page size, among them sizes that are not multiples of 16
    bytes, more pools than a launch takes, and pairs outside the pool."""
    g = torch.Generator("cuda").manual_seed(n_pools)
    shapes = [(2, 16, 64), (5,), (1,), (3, 7), (4096,), (16, 33), (2, 2, 2, 8), (1000,)]
    pools = []
    for i in range(n_pools):
        x = torch.randint(0, 256, (11, *shapes[i % len(shapes)]), generator=g, device="cuda", dtype=torch.uint8)
        if i % 5 == 1:
            x = torch.randn(11, *shapes[i % len(shapes)], generator=g, device="cuda").to(torch.bfloat16)
        if i % 5 == 2:
            x = x.view(torch.float8_e4m3fn)
        pools.append(x)
    pools[0] = torch.randint(0, 256, (11 * 30 + 1,), generator=g, device="cuda", dtype=torch.uint8)[1:].view(11, 30)
    want = [x.view(torch.uint8).clone() for x in pools]
    copies = [(0, 5), (-1, -1), (3, 7), (0, 10), (11, 2), (4, -1), (2, 11), (6, 6), (0, 1)]
    for w in want:
        for a, b in ((0, 5), (3, 7), (0, 10), (0, 1)):
            w[b] = w[a]
    paged.copy_pages(pools, int32(copies))
    for x, w in zip(pools, want):
        assert torch.equal(x.view(torch.uint8), w)
    paged.copy_pages(pools, int32(copies)[:0])
    paged.copy_pages([], int32(copies))


# ── streams, graphs ──

@gpu
def test_captured_and_on_another_stream():
    """A captured step of reserve and fork, replayed with other lengths and parents, and
    the same on a side stream behind work there."""
    rng = random.Random(8)
    B, M, page = 12, 10, 4
    lengths = [rng.randint(1, 30) for _ in range(B)]
    table, refs = random_tables(rng, B, M, page, lengths, spare=40)
    t, n, par, dt, dr = int32(lengths), int32([1] * B), int32(list(range(B))), int32(table), int32(refs)

    def step():
        plan = paged.reserve(dt, t, n, dr, page, rows=3 * B)
        t.add_(n)
        copies, missing = paged.fork(dt, t, par, dr, page)
        t.copy_(t[par.long()])
        return plan, copies, missing

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    dt.copy_(int32(table)), dr.copy_(int32(refs)), t.copy_(int32(lengths))
    for i in range(6):
        tokens = [rng.randint(0, 2) for _ in range(B)]
        parents = [rng.choice([b, b // 4 * 4]) for b in range(B)]
        n.copy_(int32(tokens)), par.copy_(int32(parents))
        if i < 4:
            graph.replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                torch.cuda._sleep(1_000_000)
                out = step()
            torch.cuda.current_stream().wait_stream(side)
        table, refs, cu, missing, places = orc.reserve(table, lengths, tokens, refs, page, 3 * B)
        lengths = [a + b for a, b in zip(lengths, tokens)]
        assert missing == 0
        table, refs, copies, _ = orc.fork(table, lengths, parents, refs, page, True)
        lengths = [lengths[x] for x in parents]
        assert dt.tolist() == table and dr.tolist() == refs and t.tolist() == lengths
        assert out[0].cu_rows.tolist() == cu and list(zip(*(x.tolist() for x in out[0][2:]))) == places
        assert [tuple(x) for x in out[1].tolist()] == copies


@gpu
def test_copies_captured_behind_anything():
    """``copy_pages`` (and ``reserve`` with many rows) as a graph's first node, behind a copy,
    behind a kernel of another library, and where two streams meet."""
    pool = torch.arange(10 * 64, device="cuda", dtype=torch.int32).view(10, 64)
    first, pairs, other = int32([[0, 3], [1, 4]]), int32([[-1, -1], [-1, -1]]), torch.zeros(64, device="cuda")
    table, refs, t, n = torch.full((2, 600), -1, dtype=torch.int32, device="cuda"), int32([0] * 1300), int32([0, 0]), int32([5000, 4000])
    paged.copy_pages([pool], pairs), paged.reserve(table, t, n, refs, 16, rows=9000)
    table.fill_(-1), refs.zero_()
    side = torch.cuda.Stream()

    def alone():
        paged.copy_pages([pool], first)

    def behind_a_copy():
        pairs.copy_(first)
        paged.copy_pages([pool], pairs)

    def behind_a_kernel():
        other.add_(1)
        paged.copy_pages([pool], first)

    def behind_two_streams():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            other.mul_(2)
        pairs.copy_(first)
        here.wait_stream(side)
        paged.copy_pages([pool], pairs)

    def reserved():
        table.fill_(-1)
        refs.zero_()
        return paged.reserve(table, t, n, refs, 16, rows=9000)

    for run in (alone, behind_a_copy, behind_a_kernel, behind_two_streams, reserved):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for i in range(3):
            pool.copy_(torch.randint(0, 1000, pool.shape, device="cuda", dtype=torch.int32))
            want = pool.clone()
            if run is not reserved:
                want[3], want[4] = want[0], want[1]
            graph.replay()
            assert torch.equal(pool, want), run.__name__
        if run is reserved:
            assert out.cu_rows.tolist() == [0, 5000, 9000] and int(refs.sum()) == 313 + 250
            assert torch.equal(out.slot, table.view(-1)[out.seq.long() * 600 + out.pos // 16] * 16 + out.pos % 16)


# ── refusals ──

@gpu
def test_refusals():
    table, t, refs = int32([[-1] * 4] * 3), int32([0, 1, 2]), int32([0] * 9)

    def no(match, table=table, t=t, x=t, refs=refs, page=8):
        for call in (lambda: paged.reserve(table, t, x, refs, page), lambda: paged.fork(table, t, x, refs, page)):
            with pytest.raises(ValueError, match=match):
                call()

    no("page_table", table=table.long())
    no("page_table", table=table[0])
    no("page_table", table=table[:1].expand(3, 4))      # rows that share their memory
    no("page_table", table=int32([[-1] * 3] * 4).t())
    no("lengths", t=t.long())
    no("lengths", t=t[:2])
    no("lengths", t=t.cpu())
    no("int32 \\[B\\]", x=t.float())
    no("int32 \\[B\\]", x=int32([1]))
    no("refs", refs=refs.view(3, 3))
    no("refs", refs=refs.cpu())
    no("page_size", page=0)
    with pytest.raises(RuntimeError, match="unsupported"):
        paged.reserve(table, t, t, refs, 2 ** 30)
    big = torch.full((8193, 1), -1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported"):
        paged.fork(big, big[:, 0].contiguous(), big[:, 0].contiguous(), refs, 8)
    with pytest.raises(ValueError, match="rows"):
        paged.reserve(table, t, t, refs, 8, rows=-1)
    x, c = torch.zeros(9, 4, device="cuda"), int32([[0, 1]])
    for pools, copies in (([x, x[1:]], c), ([x.t()], c), ([x, x.cpu()], c), ([x], c.long()), ([x], c[0]),
                          ([x[:0]], c)):
        with pytest.raises(ValueError, match="copies|pools"):
            paged.copy_pages(pools, copies)


def test_refuses_cpu_tensors():
    table, t, refs = (int32(x, "cpu") for x in ([[-1, -1]], [0], [0, 0]))
    for call in (lambda: paged.reserve(table, t, t, refs, 4), lambda: paged.fork(table, t, t, refs, 4),
                 lambda: paged.copy_pages([torch.zeros(2, 4)], int32([[0, 1]], "cpu"))):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()


def test_abi_refuses_bad_calls():
    lib, at = _capi.lib(), 1 << 20
    for fn, cls, extra in ((lib.bozo_paged_reserve, _capi.PagedReserveArgs, ("cu_rows", "missing")),
                           (lib.bozo_paged_fork, _capi.PagedForkArgs, ("parents", "copies", "missing"))):
        def status(**over):
            a = cls()
            a.batch, a.width, a.page_size, a.pages, a.table_stride = 2, 4, 16, 8, 4
            for f in ("table", "lengths", "refs", *extra):
                setattr(a, f, at)
            for f, v in over.items():
                setattr(a, f, v)
            return fn(a, None)

        assert fn(None, None) == 5
        for f in ("table", "lengths", "refs", *extra):
            assert status(**{f: None}) == 5, f
        for over, want in ((dict(batch=0), 1), (dict(width=0), 1), (dict(page_size=0), 1), (dict(pages=0), 1),
                           (dict(table_stride=-1), 1), (dict(batch=8193), 3), (dict(pages=1 << 28), 3),
                           (dict(width=1 << 28), 3)):
            assert status(**over) == want, over
        if cls is _capi.PagedReserveArgs:
            assert status(rows=-1) == 1 and status(rows=5) == 5
        else:
            assert status(copies=at + 4) == 4
    c = _capi.PagedCopyArgs()
    assert lib.bozo_paged_copy(None, None) == 5
    c.n_pools, c.n_copies = 1, 1
    assert lib.bozo_paged_copy(c, None) == 1
    c.pages = 3
    assert lib.bozo_paged_copy(c, None) == 5
    c.n_copies = 0
    assert lib.bozo_paged_copy(c, None) == 0


def test_struct_layout_matches_header(tmp_path):
    import ctypes as C
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"bozo_paged_reserve_args": _capi.PagedReserveArgs, "bozo_paged_fork_args": _capi.PagedForkArgs,
               "bozo_paged_copy_args": _capi.PagedCopyArgs, "bozo_beam_select_args": _capi.BeamSelectArgs}
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


# ── the largest ──

@gpu
def test_as_many_rows_as_there_may_be():
    rng = random.Random(11)
    B, M, page = 8192, 2, 4
    lengths = [rng.choice([-1, 0, 3, 4, 5, 8]) for _ in range(B)]
    table, refs = random_tables(rng, B, M, page, lengths, spare=12000)
    tokens = [rng.randint(0, max(0, min(4, 8 - t))) for t in lengths]
    got = check_reserve(table, lengths, tokens, refs, page, sum(tokens))
    lengths = [t + n if t >= 0 else t for t, n in zip(lengths, tokens)]
    for share in (True, False):
        parents = [rng.randrange(-1, B) for _ in range(B)]
        check_fork(got[0], lengths, parents, got[1], page, share)


@gpu
def test_a_long_row_and_a_large_pool():
    """A sequence of 2^20 tokens, and pages behind 300000 others."""
    P, page, M = 370_000, 16, 65536
    refs = [1] * 300_000 + [0, 1] * 35_000
    plan_refs, table = int32(refs), torch.full((1, M), -1, dtype=torch.int32, device="cuda")
    plan = paged.reserve(table, int32([0]), int32([35_000 * 16]), plan_refs, page, rows=1 << 20)
    free = torch.arange(300_000, P, 2, device="cuda", dtype=torch.int32)
    assert torch.equal(table[0, :35_000], free) and (table[0, 35_000:] == -1).all() and (plan_refs == 1).all()
    n = torch.arange(35_000 * 16, device="cuda")
    assert torch.equal(plan.pos[:len(n)].long(), n) and (plan.seq[:len(n)] == 0).all()
    assert torch.equal(plan.slot[:len(n)].long(), free[n // 16].long() * 16 + n % 16)
    assert (plan.seq[len(n):] == -1).all() and (plan.slot[len(n):] == -1).all() and plan.missing.item() == 0


@gpu
def test_copies_past_32_bits():
    """Pages beyond the first 2^32 bytes of a pool."""
    try:
        pool = torch.empty(5000, 1 << 20, device="cuda", dtype=torch.uint8)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("needs 5 GB of free device memory")
    pool[[0, 4997]] = torch.randint(0, 256, (2, 1 << 20), device="cuda", dtype=torch.uint8)
    keep = pool[4996].fill_(7).clone()
    paged.copy_pages([pool], int32([[0, 4999], [4997, 1]]))
    assert torch.equal(pool[4999], pool[0]) and torch.equal(pool[1], pool[4997]) and torch.equal(pool[4996], keep)
