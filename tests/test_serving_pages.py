"""A step over quantised caches does not depend on where its pages lie.

The prompts' rows are written from the same forward, bit for bit the same, whatever the pages;
the step's fp32 sums run in another order, so logits agree to 1e-4 of the largest, as a step
over fp32 caches does with the full forward.  A step that read another row, or a row's
scales from elsewhere, would be off by what a row is worth."""
import pytest
import torch

from bozo_b200 import ops, serving
from test_beam_search import ids, make, plain_matmuls  # noqa: F401 (the fixture)

gpu = pytest.mark.gpu


def step_logits(model, cache, page, scrambled):
    state = serving.PagedState(model, 4, 128, page_size=page, cache_dtype=cache)
    if scrambled:   # pages and slots that have been given back, in another order than they were taken
        slots, _ = serving.admit(state, [ids(n, n, 97) for n in (50, 3, 90, 17)])
        for slot in (slots[2], slots[0], slots[3], slots[1]):
            state.release(slot)
    slots, _ = serving.admit(state, [ids(n, n, 97) for n in (40, 7, 100)])
    feed = torch.zeros(4, dtype=torch.long, device="cuda")
    feed[slots] = torch.tensor([1, 2, 3], device="cuda")
    return serving.step(state, feed)[slots]


@gpu
@pytest.mark.parametrize("cache", [torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.int8])
def test_steps_do_not_depend_on_the_pages(cache):
    model = make("rope_global", sharp=1.0)
    want = step_logits(model, cache, 16, False)
    assert torch.isfinite(want).all()
    for page, scrambled in ((16, True), (8, True), (5, True), (1, False), (64, True)):
        got = step_logits(model, cache, page, scrambled)
        assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max()), (page, scrambled)
    ops.poll_device_error("cuda")
