"""Beam search over paged caches (``serving.BeamState``, ``serving.beam_search``): pages
reserved, shared, copied and given up on the device, the search's choices against a plain
one that runs the whole model over every hypothesis.

Scores are sums of log probabilities.  A step's logits equal the full forward's to 1e-4 of
the largest (another order of summation, as the serving tests'), so a log probability is
off by at most twice that, and a score by that for each of its tokens.  Choices between
candidates closer than that may differ: scores are compared rank by rank, and every
hypothesis' score with the full model's for its ids."""
import math

import pytest
import torch

from bozo_b200 import lm, ops, serving

gpu = pytest.mark.gpu
F4 = torch.float4_e2m1fn_x2

CFGS = {
    "rope_global": dict(vocab_size=97, dim=128, num_layers=4, num_heads=2, window=16, ffn_mult=3,
                        max_seq_len=128, dropout=0.0, use_oscillation=False, use_rope=True, global_every=2),
    "norope_osc": dict(vocab_size=97, dim=64, num_layers=2, num_heads=4, window=8, ffn_mult=3,
                       max_seq_len=96, dropout=0.0, use_oscillation=True, use_rope=False, global_every=0),
    "all_global": dict(vocab_size=61, dim=64, num_layers=2, num_heads=1, window=8, ffn_mult=2,
                       max_seq_len=80, dropout=0.0, use_oscillation=False, use_rope=True, global_every=1),
}


@pytest.fixture(autouse=True)
def plain_matmuls():
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(5)


def make(name, dtype=torch.float32, sharp=8.0):
    model = lm.TensionLM(lm.TensionConfig(**CFGS[name])).to("cuda:0", dtype).eval()
    model.lm_head.weight = torch.nn.Parameter(model.lm_head.weight.detach() * sharp)  # untied: choices far apart
    return model


def ids(n, seed, vocab):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (n,), generator=g).tolist()


@torch.no_grad()
def logp(model, seq):
    x = model(torch.tensor([seq], device="cuda:0"))[0].double()
    return torch.log_softmax(x, -1), float(x.abs().max())


def plain_search(model, prompt, beams, steps, eos):
    """(scores of the best, the largest logit met)."""
    hyps, big = [([], 0.0)], 1.0
    for _ in range(steps):
        cand = []
        for new, s in hyps:
            if new and new[-1] == eos:
                cand.append((s, new))
                continue
            lp, top = logp(model, prompt + new)
            big = max(big, top)
            best = lp[-1].topk(beams)
            cand += [(s + float(v), new + [int(t)]) for v, t in zip(best.values, best.indices)]
        hyps = [(new, s) for s, new in sorted(cand, key=lambda c: -c[0])[:beams]]
    return hyps, big


def rescored(model, prompt, new):
    lp, _ = logp(model, prompt + new)
    return sum(float(lp[len(prompt) + i - 1, t]) for i, t in enumerate(new))


@gpu
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("beams,page,graph", [(1, 16, True), (3, 5, False), (4, 16, True), (8, 1, True)])
def test_search_equals_the_plain_one(name, beams, page, graph):
    model = make(name)
    vocab = model.cfg.vocab_size
    prompts = [ids(n, n, vocab) for n in (1, 17, 30, 5)]
    steps = 12
    got = serving.beam_search(model, prompts, beams, steps, page_size=page, graph=graph, batch=3)
    for prompt, found in zip(prompts, got):
        want, big = plain_search(model, prompt, beams, steps, None)
        tol = 2e-4 * big * steps
        assert len(found) == beams and len({tuple(new) for new, _ in found}) == beams
        for (new, s), (_, ref) in zip(found, want):
            assert len(new) == steps
            assert abs(s - ref) <= tol and abs(s - rescored(model, prompt, new)) <= tol
        assert [s for _, s in found] == sorted((s for _, s in found), reverse=True)


@gpu
@pytest.mark.parametrize("graph", [False, True])
def test_ended_hypotheses_and_length_penalty(graph):
    """The most likely token of the first step ends a hypothesis: it stays among the others
    with its score while they go on; a search whose hypotheses have all ended stops."""
    model = make("rope_global")
    prompt = ids(9, 3, 97)
    for rank in (0, 1):
        eos = int(logp(model, prompt)[0][-1].topk(2).indices[rank])
        want, big = plain_search(model, prompt, 4, 20, eos)
        found = serving.beam_search(model, [prompt], 4, 20, eos=eos, graph=graph)[0]
        for (new, s), (_, ref) in zip(found, want):
            assert abs(s - ref) <= 2e-4 * big * 20
            assert eos not in new[:-1] and (len(new) == 20 or new[-1] == eos)
        assert any(new == [eos] for new, _ in found) or rank == 1
        long = serving.beam_search(model, [prompt], 4, 20, eos=eos, graph=graph, length_penalty=1.0)[0]
        by_ids = {tuple(new): s for new, s in found}
        for new, s in long:
            assert math.isclose(s, by_ids[tuple(new)] / len(new), rel_tol=1e-6)
    flat = make("rope_global", sharp=1.0)
    flat.lm_head.weight.data.zero_()                       # every token alike: token 0 first, always
    found = serving.beam_search(flat, [prompt], 1, 60, eos=0, graph=graph)[0]
    assert found[0][0] == [0] and abs(found[0][1] + math.log(97)) < 1e-5


@gpu
@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn, torch.int8, F4])
@pytest.mark.parametrize("page", [16, 8, 3])
def test_caches_in_few_bits_follow_the_hypotheses(cache, page):
    """The scores of a search over a quantised cache are those of its own ids, fed one after
    the other through a state of their own with such a cache: whatever page a hypothesis
    shares or copies holds what its own history wrote."""
    model = make("rope_global", torch.bfloat16)
    prompts = [ids(n, n, 97) for n in (23, 1)]
    beams, steps = 4, 24
    state = serving.BeamState(model, 2, beams, 23 + steps, page_size=page, cache_dtype=cache)
    for turn in range(2):                                  # the same state takes new prompts
        prompts = [[(t + turn) % 97 for t in p] for p in prompts]
        state.start(prompts)
        for _ in range(steps - 1):
            state.advance()
        refs = {g: r.cpu() for g, r in state.refs.items()}
        for g, table in state.tables.items():              # every page's count is the rows that hold it
            held = table[table >= 0].cpu().long()
            assert torch.equal(torch.bincount(held, minlength=len(refs[g])).int(), refs[g])
        ops.poll_device_error("cuda")
        for prompt, found in zip(prompts, state.results()):
            one = serving.PagedState(model, beams, 23 + steps, page_size=page, cache_dtype=cache)
            slots, logits = serving.admit(one, [prompt] * beams)
            total = torch.zeros(beams, dtype=torch.float64, device="cuda")
            for t in range(steps):
                fed = torch.tensor([new[t] for new, _ in found], device="cuda")
                lp = torch.log_softmax(logits.double(), -1)
                total += lp.gather(1, fed[:, None])[:, 0]
                big = float(logits.abs().max())
                if t + 1 < steps:
                    logits = serving.step(one, fed)
            # the same kernels on the same rows: other batch sizes of the projections move the
            # bf16 logits by a step or two (2^-8 of the largest), up to 2^-7 of it a token
            for (_, s), ref in zip(found, total.tolist()):
                assert abs(s - ref) <= steps * 2.0 ** -7 * big, (s, ref)


@gpu
@pytest.mark.parametrize("page", [16, 5])
def test_serving_on_4_bit_caches(page):
    """``PagedState`` with 4-bit pages: a step after an admitted prompt is near the full
    forward (values and keys off by at most a sixth of their sixteen's largest), a further
    turn by ``extend`` and ``generate`` run."""
    model = make("rope_global", torch.bfloat16, sharp=1.0)
    state = serving.PagedState(model, 3, 96, page_size=page, cache_dtype=F4)
    seqs = [ids(n, n, 97) for n in (20, 40, 3)]
    slots, _ = serving.admit(state, seqs)
    run = serving.PagedStepGraph(state)
    logits = run(torch.tensor([1, 2, 3], device="cuda"))
    for slot, seq, t in zip(slots, seqs, (1, 2, 3)):
        with torch.no_grad():
            ref = model(torch.tensor([seq + [t]], device="cuda"))[0, -1]
        assert float((logits[slot] - ref).abs().max()) < 0.5 * float(ref.abs().max())
    assert torch.isfinite(serving.extend(state, slots[1], ids(30, 9, 97))).all()
    out = serving.generate(model, seqs, max_new=5, cache_dtype=F4, page_size=page)
    assert [len(o) for o in out] == [25, 45, 8]


@gpu
def test_refusals():
    model = make("rope_global")
    for kw, match in ((dict(prompts=0, beams=2, max_len=20), "prompt"), (dict(prompts=1, beams=33, max_len=20), "beams"),
                      (dict(prompts=1, beams=2, max_len=129), "max_seq_len"),
                      (dict(prompts=1, beams=2, max_len=20, eos=97), "eos")):
        with pytest.raises(ValueError, match=match):
            serving.BeamState(model, **kw)
    for bad in (dict(max_new=0), dict(max_new=200)):
        with pytest.raises(ValueError, match="max_"):
            serving.beam_search(model, [[1, 2]], 2, **bad)
    state = serving.BeamState(model, 2, 2, 8)
    with pytest.raises(RuntimeError, match="start"):
        state.advance()
    for prompts in ([[1]], [[1], []], [[1], [2] * 9]):
        with pytest.raises(ValueError, match="prompts"):
            state.start(prompts)
    with pytest.raises(RuntimeError, match="together"):
        state.release(0)
    state.start([[1, 2, 3], [4] * 6])
    state.advance(), state.advance()
    with pytest.raises(ValueError, match="max_len"):
        state.advance()
    assert serving.beam_search(model, [], 2, 4) == []
    odd = lm.TensionLM(lm.TensionConfig(**dict(CFGS["norope_osc"], num_heads=8))).cuda()
    with pytest.raises(ValueError, match="multiple of 16"):
        serving.PagedState(odd, 1, 10, cache_dtype=F4)


def test_refuses_a_model_on_the_cpu():
    model = lm.TensionLM(lm.TensionConfig(**CFGS["norope_osc"]))
    with pytest.raises(RuntimeError, match="GPU"):
        serving.BeamState(model, 1, 2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        serving.PagedState(model, 1, 8, cache_dtype=F4)
