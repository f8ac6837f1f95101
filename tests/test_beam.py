"""Beam search's selection (``beam.select``) against sorting every candidate in float64.

Tokens and rows are equal: candidates of random logits are further apart than the
selection's error.  Scores: log Σ exp is a sum of V terms in fp32, each off by up to
2^-22 (the exponential) + |x − max|·2^-24·e^(x − max) ≤ 2^-24·0.4; sums of 32, then of
256 such: under 40·2^-24 relative, so 2.4e-6 + 2^-24·|score| in all."""
import math

import pytest
import torch

from bozo_b200 import _capi, beam
from oracle import paged_oracle as orc

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def check(logits, scores, done=None, eos=None):
    got = beam.select(logits, scores, done=done, eos=eos)
    want = orc.select(logits.cpu(), scores.cpu(), None if done is None else done.cpu(), eos)
    assert got[0].dtype == F32 and got[1].dtype == torch.int64 and got[2].dtype == torch.int32
    s, ref = got[0].cpu().double(), want[0]
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(s), fin)
    assert bool(((s - ref)[fin].abs() <= 2.4e-6 + 2.0 ** -24 * ref[fin].abs()).all())
    assert (s[~fin] == -math.inf).all()
    assert torch.equal(got[1].cpu(), want[1]), (got[1], want[1])
    assert torch.equal(got[2].cpu(), want[2])
    return got


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,K,V", [(1, 1, 1), (1, 4, 97), (3, 2, 8192), (2, 5, 8193), (5, 8, 2048), (1, 32, 32),
                                   (2, 32, 40000), (64, 4, 513), (1, 3, 262147), (7, 1, 16385), (1, 16, 32768)])
def test_random_logits(dtype, N, K, V):
    logits = (torch.randn(N * K, V, device="cuda") * 3).to(dtype)
    check(logits, -20 * torch.rand(N, K, device="cuda"))


@gpu
@pytest.mark.parametrize("K", [2, 4, 9])
def test_first_step_and_ended_hypotheses(K):
    N, V = 3, 5000
    logits = torch.randn(N * K, V, device="cuda")
    first = torch.full((N, K), -math.inf, device="cuda")
    first[:, 0] = 0
    _, _, rows = check(logits, first)
    assert (rows % K == 0).all()
    done = torch.zeros(N, K, dtype=torch.bool, device="cuda")
    done[0, 1] = done[1] = True
    scores = -torch.rand(N, K, device="cuda")
    s, t, r = check(logits, scores, done, 17)
    assert torch.equal(s[1], scores[1].sort(descending=True)[0]) and (t[1] == 17).all()
    check(logits, scores, done, 0)
    check(logits, scores, done, V - 1)
    check(logits, first, done, 3)
    check(logits, scores, torch.zeros_like(done), 3)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ties_go_to_the_lowest(dtype):
    """Equal logits in a row, equal rows, all of them equal, ±0."""
    N, K, V = 2, 4, 9000
    logits = torch.randint(-2, 3, (N * K, V), device="cuda").to(dtype)
    check(logits, -torch.rand(N, K, device="cuda"))
    same = logits[:1].expand(N * K, V).contiguous()
    check(same, torch.zeros(N, K, device="cuda"))
    check(torch.zeros(N * K, V, device="cuda", dtype=dtype), torch.zeros(N, K, device="cuda"))
    zeros = torch.zeros(N * K, V, device="cuda", dtype=dtype)
    zeros[:, ::2] = -0.0
    check(zeros, torch.zeros(N, K, device="cuda"))
    check(zeros[:, :K], torch.zeros(N, K, device="cuda"))
    few = torch.zeros(3 * 20, 70001, device="cuda", dtype=dtype)   # several tiles of equal logits, K of them better
    few[:, 5000::3001] = 1
    check(few, torch.zeros(3, 20, device="cuda"))
    check(few[:3], torch.zeros(3, 1, device="cuda"))


@gpu
@pytest.mark.parametrize("V", [50, 20000])
def test_masked_tokens_and_rows_that_are_not_finite(V):
    """Tokens masked by −inf or the type's lowest value, all but a few, all; NaN, +inf;
    scores that are not finite: those are worth −inf and come last, lowest first."""
    K = 6
    logits = torch.randn(3 * K, V, device="cuda")
    logits[:, 5:] = -math.inf                       # fewer tokens than the hypotheses want
    logits[1] = -math.inf
    logits[2, V // 2] = math.nan
    logits[3, 7] = math.inf
    logits[4, :] = torch.finfo(F32).min
    logits[K:2 * K] = -math.inf                      # a prompt with nothing
    logits[2 * K:] = torch.finfo(F32).min
    logits[2 * K + 1, 3] = 4.0
    scores = -torch.rand(3, K, device="cuda")
    for bad in (None, math.inf, -math.inf, math.nan):
        if bad is not None:
            scores[2, 1] = scores[0, 0] = bad
        got = beam.select(logits, scores)
        want = orc.select(logits.cpu(), scores.cpu(), None, None)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
        fin = want[0] > -1e30
        assert ((got[0].cpu().double() - want[0])[fin].abs() < 1e-5).all()
        assert not torch.isnan(got[0]).any()
    done = torch.ones(3, K, dtype=torch.bool, device="cuda")
    check(logits.nan_to_num(0, 0, -math.inf), scores.nan_to_num(-1, -1, -1), done, V - 2)


@gpu
@pytest.mark.parametrize("shift", [-300.0, 300.0])
def test_logits_far_from_zero(shift):
    """All logits below the smallest exponential, or above the largest, in rows that leave
    most threads without one."""
    for V in (9, 5000, 40001):
        check(torch.randn(8, V, device="cuda") + shift, -torch.rand(2, 4, device="cuda"))


@gpu
def test_strided_rows_and_unaligned_ones():
    x = torch.randn(8, 3001, device="cuda", dtype=BF16)
    check(x[:, 1:], -torch.rand(2, 4, device="cuda"))
    check(x[::2, 3:2999], -torch.rand(1, 4, device="cuda"))
    flat = torch.randn(5 * 9001 + 16, device="cuda")
    for dtype in (F32, F16):
        for first in range(9):
            for V in (5, 64, 8190):
                y = flat.to(dtype)[first:first + 4 * 9001].view(4, 9001)[:, :V]
                check(y, -torch.rand(1, 4, device="cuda"))
    one = torch.randn(1, 3001, device="cuda").expand(4, 3001)   # a prompt's logits for all its hypotheses
    first = torch.tensor([[0.0] + [-math.inf] * 3], device="cuda")
    check(one, first)


@gpu
def test_captured_on_another_stream_and_twice_at_once():
    a, b = torch.randn(8, 9001, device="cuda"), torch.randn(8, 9001, device="cuda")
    sa, sb = -torch.rand(2, 4, device="cuda"), -torch.rand(1, 8, device="cuda")
    want = [beam.select(a, sa), beam.select(b, sb)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        one = beam.select(a, sa)
        with torch.cuda.stream(side):
            two = beam.select(b, sb)
        torch.cuda.synchronize()
        for g, w in zip((one, two), want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam.select(a, sa)
    a.normal_(), sa.uniform_(-3, 0)
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, beam.select(a, sa)))


@gpu
def test_refusals():
    x, s = torch.randn(8, 64, device="cuda"), torch.zeros(2, 4, device="cuda")
    done = torch.zeros(2, 4, dtype=torch.bool, device="cuda")

    def no(error, match, *a, **kw):
        with pytest.raises(error, match=match):
            beam.select(*a, **kw)

    no(ValueError, "logits", x[:7], s)
    no(ValueError, "logits", x.t().contiguous().t(), s)
    no(ValueError, "scores", x, s.double())
    no(ValueError, "scores", x, s.cpu())
    no(ValueError, "scores", x, s.view(-1))
    no(ValueError, "beams", x[:, :3], s)
    no(ValueError, "beams", torch.randn(33, 64, device="cuda"), torch.zeros(1, 33, device="cuda"))
    no(ValueError, "eos", x, s, done=done)
    no(ValueError, "eos", x, s, done=done, eos=64)
    no(ValueError, "eos", x, s, eos=-2)
    no(ValueError, "done", x, s, done=done.int(), eos=1)
    no(ValueError, "done", x, s, done=done[:1], eos=1)
    no(TypeError, "dtype", x.double(), s)
    no(RuntimeError, "no gradient", x.clone().requires_grad_(), s)


def test_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA only"):
        beam.select(torch.zeros(2, 8), torch.zeros(1, 2))


def test_abi_refuses_bad_calls():
    lib, at = _capi.lib(), 1 << 20

    def status(**over):
        a = _capi.BeamSelectArgs()
        a.prompts, a.beams, a.vocab, a.row_stride, a.eos = 2, 4, 100, 100, -1
        for f in ("logits", "scores", "out_scores", "out_tokens", "out_rows"):
            setattr(a, f, at)
        for f, v in over.items():
            setattr(a, f, v)
        return lib.bozo_beam_select(a, None)

    for over, want in ((dict(prompts=0), 1), (dict(beams=0), 1), (dict(vocab=3), 1), (dict(row_stride=-1), 1),
                       (dict(eos=100), 1), (dict(done=at), 1), (dict(dtype=3), 2), (dict(beams=33), 3),
                       (dict(vocab=(1 << 20) + 1), 3), (dict(prompts=20000), 3), (dict(logits=None), 5),
                       (dict(out_rows=None), 5)):
        assert status(**over) == want, over
    assert lib.bozo_beam_select(None, None) == 5


def test_oracle_by_hand():
    x = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.6, 0.3]]))
    s, t, r = orc.select(x, torch.log(torch.tensor([[0.4, 0.5]])), None, None)
    assert t.tolist() == [[1, 0]] and r.tolist() == [[1, 0]]
    assert torch.allclose(torch.exp(s), torch.tensor([[0.3, 0.2]], dtype=torch.float64), atol=1e-6)


@gpu
def test_logits_past_32_bits():
    """More than 2^32 bytes of logits: the last prompts' rows."""
    N, K, V = 9000, 4, 65536
    try:
        logits = torch.empty(N * K, V, device="cuda", dtype=BF16)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("needs 5 GB of free device memory")
    scores = torch.full((N, K), -math.inf, device="cuda")   # only the last ones are read
    logits[-3 * K:] = torch.randn(3 * K, V, device="cuda").to(BF16)
    scores[-3:] = -torch.rand(3, K, device="cuda")
    s, t, r = beam.select(logits, scores)
    want = beam.select(logits[-3 * K:].clone(), scores[-3:].clone())
    assert torch.equal(s[-3:], want[0]) and torch.equal(t[-3:], want[1])
    assert torch.equal(r[-3:], want[2] + (N - 3) * K)
    assert (s[:-3] == -math.inf).all() and torch.equal(t[0], torch.arange(K, device="cuda"))
