"""Serving over paged caches (``bozo_b200.serving``): every sequence of a batch
whose members come, grow, go on and leave at their own times gets the logits
(and τ rows) of a full forward over its own ids.  Tolerances as the ring-cache
decode tests' (fp32, another order of summation); 8-bit caches are compared
with a model of the rounding in ``test_paged.py``, here with the logits' scale."""
import pytest
import torch

from bozo_b200 import lm, ops, serving

gpu = pytest.mark.gpu

CFGS = {
    "rope_global": dict(vocab_size=97, dim=128, num_layers=4, num_heads=2, window=16, ffn_mult=3,
                        max_seq_len=192, dropout=0.0, use_oscillation=False, use_rope=True,
                        global_every=2),
    "norope_osc": dict(vocab_size=97, dim=64, num_layers=2, num_heads=4, window=8, ffn_mult=3,
                       max_seq_len=96, dropout=0.0, use_oscillation=True, use_rope=False,
                       global_every=0),
}


@pytest.fixture(autouse=True)
def plain_matmuls():
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(5)


def make(name, dtype=torch.float32):
    return lm.TensionLM(lm.TensionConfig(**CFGS[name])).to("cuda:0", dtype).eval()


def ids(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 97, (n,), generator=g).tolist()


@torch.no_grad()
def full(model, seq, export=False):
    res = model(torch.tensor([seq], device="cuda:0"), return_all=export)
    return (res[0][0, -1], [t[0, -1] for t in res[2]]) if export else res[0, -1]


def close(got, ref, what, tol=1e-4):
    scale = float(ref.abs().max())
    torch.testing.assert_close(got, ref, rtol=tol, atol=tol * scale, msg=lambda m: f"{what}: {m}")


@gpu
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("page,graph,export", [(16, False, False), (16, True, True), (5, True, False),
                                               (32, False, True)])
def test_sequences_come_grow_and_go(name, page, graph, export):
    model = make(name)
    state = serving.PagedState(model, 4, 96, page_size=page)
    run = serving.PagedStepGraph(state, export=export) if graph else (
        lambda tok: serving.step(state, tok, export=export))
    held = {}

    def admit(*lens):
        prompts = [ids(n, 10 * n + len(held)) for n in lens]
        slots, logits = serving.admit(state, prompts)
        for s, p, row in zip(slots, prompts, logits):
            held[s] = list(p)
            close(row, full(model, p), f"prompt of {len(p)}")

    def steps(n, seed):
        for i in range(n):
            new = ids(state.slots, seed + i)
            res = run(torch.tensor(new, device="cuda:0"))
            logits, taus = res if export else (res, None)
            for s in held:
                held[s].append(new[s])
                if export:
                    ref, rows = full(model, held[s], True)
                    close(logits[s], ref, f"slot {s} at {len(held[s])}")
                    for got, want in zip(taus, rows):
                        w = min(got.shape[-1], want.shape[-1])
                        torch.testing.assert_close(got[s, :, :w], want[:, :w], rtol=1e-4, atol=1e-5)
                else:
                    close(logits[s], full(model, held[s]), f"slot {s} at {len(held[s])}")

    def leave(s):
        state.release(s)
        del held[s]

    admit(1, 37, 16)
    steps(3, 100)
    leave(1)
    admit(5, 50)
    steps(4, 200)
    leave(0)
    steps(2, 300)
    for s, n in ((2, 1), (3, 21)):
        if s in held:
            new = ids(n, 400 + s)
            held[s] += new
            if export:  # a further turn is a plain forward (count normalisation in local layers)
                continue
            close(serving.extend(state, s, new), full(model, held[s]), f"slot {s} extended by {n}")
    if not export:
        steps(3, 500)
        assert [state.length(s) for s in held] == [len(v) for v in held.values()]
    ops.poll_device_error("cuda:0")


@gpu
@pytest.mark.parametrize("chunk", [1, 7, 16, 40])
def test_a_sequence_extended_in_chunks(chunk):
    """Chunks shorter and longer than the window and its ring."""
    model = make("rope_global")
    state = serving.PagedState(model, 2, 192, page_size=16)
    seq = ids(3, 1)
    (slot,), _ = serving.admit(state, [seq])
    for i in range(100 // chunk if chunk > 1 else 30):
        new = ids(chunk, 50 + i)
        seq += new
        close(serving.extend(state, slot, new), full(model, seq), f"{len(seq)} ids in chunks of {chunk}")


@gpu
def test_past_max_seq_len_the_oldest_keys_leave():
    """Global layers reach their table's pages: the same as the ring caches of
    ``decode`` with that capacity, every step."""
    from bozo_b200 import decode
    model = make("rope_global")
    model.cfg.max_seq_len = 32
    seq = ids(30, 3)
    state = serving.PagedState(model, 2, 120, page_size=16)
    ring = decode.DecodeState(model, 1, 120)
    (slot,), a = serving.admit(state, [seq])
    b = decode.prefill(ring, torch.tensor([seq], device="cuda:0"))
    close(a[0], b[0], "prompt")
    for i in range(60):
        tok = torch.tensor(ids(2, 900 + i), device="cuda:0")
        close(serving.step(state, tok)[slot], decode.step(ring, tok[slot:slot + 1])[0], f"step {i}")


@gpu
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.int8, torch.bfloat16])
def test_smaller_caches(cache):
    """e4m3 holds 4 bits of significand, int8 8 bits of the row's largest: the
    logits follow the exact ones within a few of those roundings."""
    model = make("rope_global")
    state = serving.PagedState(model, 3, 96, cache_dtype=cache)
    seqs = [ids(n, n) for n in (20, 64, 41)]
    slots, _ = serving.admit(state, seqs)
    tol = {torch.float8_e4m3fn: 2.0 ** -4, torch.int8: 2.0 ** -6, torch.bfloat16: 2.0 ** -7}[cache]
    for i in range(8):
        new = ids(3, 70 + i)
        logits = serving.step(state, torch.tensor(new, device="cuda:0"))
        for s, seq in zip(slots, seqs):
            seq.append(new[s])
            ref = full(model, seq)
            err = float((logits[s] - ref).norm() / ref.norm())
            assert err <= tol, (cache, i, err)
    seqs[1] += ids(9, 99)
    got, ref = serving.extend(state, slots[1], seqs[1][-9:]), full(model, seqs[1])
    assert float((got - ref).norm() / ref.norm()) <= tol


@gpu
def test_generate_equals_one_prompt_at_a_time():
    """Greedy in effect (temperature near zero): continuous batching over 3 slots
    gives each prompt what it gets alone."""
    from bozo_b200 import decode
    model = make("rope_global")
    prompts = [ids(n, n) for n in (4, 30, 17, 1, 55, 8)]
    got = serving.generate(model, prompts, max_new=9, temp=1e-4, slots=3)
    for p, g in zip(prompts, got):
        assert g == decode.generate(model, p, max_new=9, temp=1e-4)
    assert serving.generate(model, prompts[:2], max_new=0) == prompts[:2]
    eager = serving.generate(model, prompts, max_new=9, temp=1e-4, slots=2, graph=False, page_size=7)
    assert eager == got


@gpu
def test_pages_run_out_and_come_back():
    model = make("rope_global")
    state = serving.PagedState(model, 3, 64, page_size=16, pages=4)
    a, _ = serving.admit(state, [ids(30, 1)])       # two pages
    with pytest.raises(RuntimeError, match="out of pages"):
        serving.admit(state, [ids(40, 2)])          # three
    assert state.free_pages == 2 and state.idle == [1, 2]
    b, _ = serving.admit(state, [ids(32, 2)])
    assert state.free_pages == 0
    before = [state.length(a[0]), state.length(b[0])]
    with pytest.raises(RuntimeError, match="out of pages"):
        serving.step(state, torch.zeros(3, dtype=torch.long, device="cuda:0"))
    assert [state.length(a[0]), state.length(b[0])] == before and state.free_pages == 0
    state.release(a[0])
    assert state.free_pages == 2
    seq = ids(32, 2) + [7]
    logits = serving.step(state, torch.full((3,), 7, dtype=torch.long, device="cuda:0"))
    close(logits[b[0]], full(model, seq), "after a release")
    ops.poll_device_error("cuda:0")


@gpu
def test_refusals():
    model = make("norope_osc")
    with pytest.raises(ValueError, match="learned positions"):
        serving.PagedState(model, 1, 97)
    with pytest.raises(ValueError, match="at least 1"):
        serving.PagedState(model, 0, 8)
    state = serving.PagedState(model, 2, 20)
    for bad in ([], [[]], [[1] * 97]):
        with pytest.raises(ValueError):
            serving.admit(state, bad)
    with pytest.raises(ValueError, match="max_len"):
        serving.admit(state, [[1] * 21])
    with pytest.raises(RuntimeError, match="idle slots"):
        serving.admit(state, [[1], [2], [3]])
    with pytest.raises(ValueError, match="idle"):
        state.release(0)
    with pytest.raises(ValueError, match="idle"):
        serving.extend(state, 1, [3])
    (s,), _ = serving.admit(state, [[1] * 20])
    with pytest.raises(ValueError, match="max_len"):
        serving.step(state, torch.zeros(2, dtype=torch.long, device="cuda:0"))
    with pytest.raises(ValueError, match="max_len"):
        serving.extend(state, s, [1])
    with pytest.raises(ValueError, match="at least one"):
        serving.extend(state, s, [])
    with pytest.raises(ValueError, match="tokens must be"):
        serving.step(state, torch.zeros(3, dtype=torch.long, device="cuda:0"))


def test_serving_needs_a_gpu_model():
    model = lm.TensionLM(lm.TensionConfig(**CFGS["norope_osc"]))
    with pytest.raises(RuntimeError, match="GPU"):
        serving.PagedState(model, 1, 16)
