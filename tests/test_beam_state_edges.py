"""``serving.BeamState`` and ``serving.beam_search`` at their edges: calls that a beam search's
state does not serve, failed calls, and what is held after its pages move."""
import pytest
import torch

from bozo_b200 import serving
from test_beam_search import ids, make, plain_matmuls  # noqa: F401 (the fixture)

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
