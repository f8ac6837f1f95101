"""``serving.BeamState`` and ``serving.beam_search`` at their edges: calls that a beam search's
state does not serve, failed calls, and what is held after its pages move."""
import pytest
import torch

from bozo_b200 import ops, paged, serving
from test_beam_search import CFGS, ids, make, plain_matmuls  # noqa: F401 (the fixture)

gpu = pytest.mark.gpu


def held(state):
    """Everything a state holds on the device."""
    return ([state.local_table, state.global_table, state.lengths, state.tokens, state.scores, state.chosen, state.steps]
            + list(state.refs.values()) + [p for pools in state.pools.values() for p in pools])


@gpu
@pytest.mark.parametrize("name", ["rope_global", "norope_osc"])   # with and without global layers
def test_calls_for_single_slots_are_refused(name):
    """The pages of a beam search are counted on the device: what counts them on the host
    (``admit``, ``extend``, ``step``, ``PagedStepGraph``, ``release`` and the queries beside them)
    would hand out pages that hypotheses hold.  It is refused, and changes nothing."""
    model = make(name)
    state = serving.BeamState(model, 2, 3, 40, graph=False)
    for started in (False, True):
        if started:
            state.start([ids(7, 1, 60), ids(20, 2, 60)])
            state.advance()
        before = [x.clone() for x in held(state)]
        feed = torch.zeros(6, dtype=torch.long, device="cuda")
        for call in (lambda: serving.admit(state, [[1, 2, 3]]), lambda: serving.extend(state, 0, [1]),
                     lambda: serving.step(state, feed), lambda: serving.PagedStepGraph(state),
                     lambda: state.release(0), lambda: state.length(0), lambda: state.idle, lambda: state.free_pages):
            with pytest.raises(RuntimeError, match="together"):
                call()
        assert all(torch.equal(a, b) for a, b in zip(held(state), before))
    state.advance()


@gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_state_without_prompts_has_nothing_to_say(graph, monkeypatch):
    """Before ``start``, and after a call that failed midway, there is nothing to advance or to
    return; refused prompts leave the running search as it was."""
    model = make("rope_global")
    state = serving.BeamState(model, 2, 3, 40, graph=graph)
    prompts = [ids(7, 1, 60), ids(20, 2, 60)]

    def empty():
        for call in (state.advance, state.results, lambda: state.results(1.0)):
            with pytest.raises(RuntimeError, match="start"):
                call()

    empty()
    state.start(prompts)
    state.advance()
    want = state.results()
    with pytest.raises(ValueError, match="prompts"):
        state.start(prompts[:1])
    assert state.results() == want

    def fails(*args):
        raise MemoryError("no room")

    with monkeypatch.context() as m:
        m.setattr(serving, "_prefill", fails)
        with pytest.raises(MemoryError):
            state.start(prompts)
    empty()
    state.start(prompts)
    state.advance()
    assert state.results() == want
    if not graph:
        with monkeypatch.context() as m:
            m.setattr(serving.paged, "copy_pages", fails)      # tables moved, pages not
            with pytest.raises(MemoryError):
                state.advance()
        empty()
        state.start(prompts)
        state.advance()
        assert state.results() == want


@gpu
def test_more_hypotheses_than_a_table_has_rows_are_refused():
    """Before anything is held: the table's kernels refused it, in the middle of start()."""
    model = make("all_global")
    for prompts, beams in ((8193, 1), (2049, 4), (257, 32)):
        with pytest.raises(ValueError, match="8192"):
            serving.BeamState(model, prompts, beams, 8, graph=False)


@gpu
def test_search_refuses_batches_of_nothing():
    model = make("all_global")
    for batch in (0, -1, -16):                     # −1 returned no result for any prompt
        with pytest.raises(ValueError, match="batch must be at least 1"):
            serving.beam_search(model, [[1, 2], [3]], 2, 4, batch=batch)


@gpu
@pytest.mark.parametrize("name,bounded", [("rope_global", True), ("norope_osc", True), ("rope_local", False)])
def test_long_prompts_keep_their_last_ids(name, bounded, monkeypatch):
    """The last id that is fed takes the last position: max_seq_len − max_new + 1 ids of the
    prompt where positions are bounded, max_seq_len else."""
    monkeypatch.setitem(CFGS, "rope_local", dict(CFGS["rope_global"], global_every=0))
    model = make(name)
    limit, vocab, steps = model.cfg.max_seq_len, model.cfg.vocab_size, 6
    keep = limit - steps + 1 if bounded else limit
    taken, start = [], serving.BeamState.start
    monkeypatch.setattr(serving.BeamState, "start", lambda self, p: (taken.append(p), start(self, p))[1])
    prompts = [ids(n, n, vocab) for n in (limit + 9, keep, keep + 1, 5)]
    found = serving.beam_search(model, prompts, 2, steps, graph=False)
    assert taken == [[p[-keep:] for p in prompts]] and all(len(new) == steps for f in found for new, _ in f)


def cached_rows(state, lengths):
    """Each slot's cached rows as they are held, a list of (k, v) by layer and slot: the last ones
    that the layer's pages reach."""
    res = []
    for li, lay in enumerate(state.layers):
        table = state.table(li)
        counts = [min(max(t, 0), table.shape[1] * state.page_size) for t in lengths]
        cu = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
        start = torch.tensor([t - n if t >= 0 else -1 for t, n in zip(lengths, counts)], dtype=torch.int32, device="cuda")
        k, v = paged.read_kv(lay.k, lay.v, table, start, cu, sum(counts), dtype=torch.float32, **lay.scales)
        res.append(list(zip(k.split(counts), v.split(counts))))
    return res


@gpu
@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn, torch.int8, torch.float4_e2m1fn_x2])
@pytest.mark.parametrize("page", [16, 8, 3])
def test_every_hypothesis_holds_its_parents_rows(cache, page):
    """What a hypothesis' pages hold after they were shared, moved and copied is what its parent's
    held before, bit for bit, in every layer: codes, scales and group scales."""
    model = make("rope_global", torch.bfloat16, sharp=2.0)
    state = serving.BeamState(model, 2, 5, 23 + 40, page_size=page, cache_dtype=cache, graph=False)
    choose, forks = state._choose, []

    def watched(logits):
        lengths = state.lengths.tolist()
        before = cached_rows(state, lengths)
        choose(logits)
        parents = state.chosen[int(state.steps) - 1, 1].tolist()
        lengths = [lengths[x] for x in parents]
        assert state.lengths.tolist() == lengths
        for li, (was, now) in enumerate(zip(before, cached_rows(state, lengths))):
            for r, x in enumerate(parents):
                for a, b in zip(was[x], now[r]):
                    assert torch.equal(a.view(torch.int32), b.view(torch.int32)), (li, r, x)
        forks.append(len(set(parents)) < len(parents))

    state._choose = watched
    state.start([ids(23, 1, 97), ids(2, 2, 97)])
    for _ in range(40):
        state.advance()
    assert len(forks) == 41 and sum(forks) > 20
    ops.poll_device_error("cuda")
