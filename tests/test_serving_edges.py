"""Serving over paged caches (``bozo_b200.serving``) at its limits: sequences longer
than a global layer's reach, and calls that are refused."""
import pytest
import torch

from bozo_b200 import decode, ops, serving
from test_serving import close, full, ids, make

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def plain_matmuls():
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(5)


@gpu
@pytest.mark.parametrize("chunks", [(1, 1, 1, 7), (3, 9, 1, 20), (40, 1, 5), (64, 2), (2, 31, 33)])
def test_a_sequence_extended_past_the_reach(chunks):
    """A global layer attends the last C keys, however the ids came: the same logits
    as the same ids fed one by one, in chunks that end before, cross and begin past C,
    and the same steps after them."""
    model = make("rope_global")
    model.cfg.max_seq_len = 32
    one = serving.PagedState(model, 2, 120, page_size=16)
    many = serving.PagedState(model, 2, 120, page_size=16)
    first = ids(30, 8)
    (a,), _ = serving.admit(one, [first])
    (b,), _ = serving.admit(many, [first])
    for i, n in enumerate(chunks):
        new = ids(n, 40 + i)
        for x in new:
            want = serving.step(one, torch.full((2,), x, dtype=torch.long, device="cuda:0"))[a]
        close(serving.extend(many, b, new), want, f"{n} ids from {one.length(a) - n} on")
    assert one.length(a) == many.length(b)
    for i in range(3):
        tok = torch.tensor(ids(2, 90 + i), device="cuda:0")
        close(serving.step(many, tok)[b], serving.step(one, tok)[a], f"step {i} after")
    ops.poll_device_error("cuda:0")


@gpu
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.int8])
def test_extended_past_the_reach_of_an_8_bit_cache(cache):
    """As above; the keys of a chunk that lies past C are attended as the cache holds
    them, so a chunk of any length gives what the same ids give one by one."""
    model = make("rope_global")
    model.cfg.max_seq_len = 32
    one, many = (serving.PagedState(model, 1, 100, page_size=16, cache_dtype=cache) for _ in range(2))
    first = ids(32, 8)
    for s in (one, many):
        serving.admit(s, [first])
    new = ids(9, 3)
    for x in new:
        want = serving.step(one, torch.tensor([x], device="cuda:0"))[0]
    got = serving.extend(many, 0, new)
    # local layers attend a chunk's own keys before they are rounded to 8 bits
    tol = {torch.float8_e4m3fn: 2.0 ** -4, torch.int8: 2.0 ** -6}[cache]
    assert float((got - want).norm() / want.norm()) <= tol


@gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_refused_step_changes_nothing(graph):
    """Tokens of a wrong shape, type or device: refused before any page is taken or
    a length advanced."""
    model = make("rope_global")
    state = serving.PagedState(model, 2, 64, page_size=16)
    (s,), _ = serving.admit(state, [ids(16, 1)])           # the next token takes a page
    run = serving.PagedStepGraph(state) if graph else (lambda tok: serving.step(state, tok))
    free, held = state.free_pages, state.length(s)
    for bad in (torch.zeros(1, dtype=torch.long, device="cuda:0"), torch.zeros((), dtype=torch.long, device="cuda:0"),
                torch.zeros(3, dtype=torch.long, device="cuda:0"), torch.zeros(2, 1, dtype=torch.long, device="cuda:0"),
                torch.zeros(2, dtype=torch.float32, device="cuda:0"), torch.zeros(2, dtype=torch.bool, device="cuda:0"),
                *([] if graph else [torch.zeros(2, dtype=torch.long)])):  # a replay copies tokens from any device
        with pytest.raises((ValueError, TypeError), match="tokens"):
            run(bad)
        assert (state.free_pages, state.length(s)) == (free, held)
        assert state.lengths.tolist()[s] == held
    seq = ids(16, 1) + [7]
    got = run(torch.full((2,), 7, dtype=torch.long, device="cuda:0"))
    close(got[s], full(model, seq), "after the refusals")
    seq.append(9)
    got = run(torch.full((2,), 9, dtype=torch.int16, device="cuda:0"))
    close(got[s], full(model, seq), "tokens of another integer type")


@gpu
def test_a_failed_step_advances_no_length(monkeypatch):
    """A step that ends in an exception leaves the host's and the device's lengths
    alike, and the next one gives what it would have given."""
    model = make("rope_global")
    state = serving.PagedState(model, 2, 64, page_size=16)
    (s,), _ = serving.admit(state, [ids(16, 1)])
    tok = torch.full((2,), 7, dtype=torch.long, device="cuda:0")

    def fail(*a, **kw):
        raise torch.OutOfMemoryError("out of memory")

    with monkeypatch.context() as m:
        m.setattr(model.final_norm, "forward", fail)
        with pytest.raises(torch.OutOfMemoryError):
            serving.step(state, tok)
    assert state.length(s) == state.lengths.tolist()[s] == 16
    close(serving.step(state, tok)[s], full(model, ids(16, 1) + [7]), "the next step")
    state.release(s)
    assert state.free_pages == 8


@gpu
@pytest.mark.parametrize("page", [5, 7, 24])
def test_past_max_seq_len_global_layers_reach_whole_pages(page):
    """A page size that does not divide max_seq_len: the reach is that of a ring of
    so many whole pages."""
    model = make("rope_global")
    model.cfg.max_seq_len = 32
    state = serving.PagedState(model, 2, 100, page_size=page)
    model.cfg.max_seq_len = state.global_table.shape[1] * page
    ring = decode.DecodeState(model, 1, 100)
    seq = ids(30, 3)
    (slot,), a = serving.admit(state, [seq])
    close(a[0], decode.prefill(ring, torch.tensor([seq], device="cuda:0"))[0], "prompt")
    for i in range(25):
        tok = torch.tensor(ids(2, 700 + i), device="cuda:0")
        close(serving.step(state, tok)[slot], decode.step(ring, tok[slot:slot + 1])[0], f"step {i}")


@gpu
def test_a_failed_capture_leaves_the_sequences(monkeypatch):
    model = make("rope_global")
    state = serving.PagedState(model, 2, 64, page_size=16)
    (s,), _ = serving.admit(state, [ids(16, 1)])

    def fail(*a, **kw):
        raise torch.OutOfMemoryError("out of memory")

    with monkeypatch.context() as m:
        m.setattr(model.final_norm, "forward", fail)
        with pytest.raises(torch.OutOfMemoryError):
            serving.PagedStepGraph(state)
    assert state.lengths.tolist()[s] == 16
    run = serving.PagedStepGraph(state)
    close(run(torch.full((2,), 7, dtype=torch.long, device="cuda:0"))[s], full(model, ids(16, 1) + [7]), "a step")
