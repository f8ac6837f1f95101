"""Beam search's selection at its largest sizes, and how far its logarithms may be off."""
import math

import pytest
import torch

from bozo_b200 import beam

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def log_error(V):
    """Bound of log Σ exp's error.  In units of 2^-24 of the sum: 4 for the exponential of a term
    (2^-22); (x − ref)·log2 e rounded three times, 2.3 · (m − x), which over the sum's terms is at
    most 2.3 (ln V + ¼) on average (their entropy is); 18 additions of a batch; the thread's
    sum keeps what its additions leave over, but where its reference rises, by ¼ or more, it is
    multiplied by an exponential, 5, of which a row of rises adds 1 / (1 − e^-¼) = 4.5; 1 for the
    two parts' sum; thread to warp, warp to block and part to row an exponential and a product
    each, 15; their 5 + 5 + 7 additions.  The logarithm itself 1.4e-9."""
    return (4 + 18 + 22.5 + 1 + 15 + 17 + 2.3 * (math.log(V) + 0.25)) * 2.0 ** -24 + 1.4e-9


def check(logits, scores):
    """Scores are those of the tokens returned, and the K best, both to the logarithm's error."""
    N, K = scores.shape
    s, t, r = beam.select(logits, scores)
    lse = torch.stack([torch.logsumexp(x.double(), -1) for x in logits])
    worth = lambda rows, x: scores.view(-1).double()[rows] + x - lse[rows]
    rows = r.long()
    got = worth(rows, logits[rows, t].double())
    tol = log_error(logits.shape[1])
    assert bool(((s.double() - got).abs() <= tol + 2.0 ** -24 * got.abs()).all()), float((s.double() - got).abs().max())
    best = torch.stack([x.double().topk(K)[0] for x in logits])
    all_ = worth(torch.arange(N * K, device="cuda")[:, None], best).view(N, K * K)
    want = all_.sort(descending=True)[0][:, :K]
    assert bool(((got - want).abs() <= 2 * tol).all())
    assert ((rows // K) == torch.arange(N, device="cuda")[:, None]).all()


@gpu
@pytest.mark.parametrize("V,N,K,dtype", [
    (1 << 20, 64, 2, F32),      # more than 100 batches a thread
    (1 << 20, 5, 3, BF16), ((1 << 20) - 3, 3, 32, F16), (1 << 20, 1, 1, F32), (1 << 20, 2, 4, F32),
    (50257, 32, 8, BF16), (32768, 64, 8, F32), (8191, 2, 1, F32)])
def test_logarithms_of_long_rows(V, N, K, dtype):
    n = N * K
    scores = -torch.rand(N, K, device="cuda")
    base = torch.arange(V, device="cuda", dtype=F32)
    rows = {
        "random": torch.randn(n, V, device="cuda") * 3,
        "most of the sum far below the largest": torch.randn(n, V, device="cuda") * 1e-2 - (math.log(V) - 0.2),
        "rising slowly": (base / V * 0.01).repeat(n, 1) + torch.randn(n, V, device="cuda") * 1e-4,
        "rising": (base / V * 14).repeat(n, 1) + torch.randn(n, V, device="cuda") * 1e-4,
        "falling": (base / V * -14).repeat(n, 1) + torch.randn(n, V, device="cuda") * 1e-4,
    }
    rows["most of the sum far below the largest"][:, 5] = 0
    for what, x in list(rows.items()):
        check(x.to(dtype), scores)
        del rows[what], x


@gpu
def test_the_logarithm_itself():
    """Rows of n equal logits, the rest masked: the sum is n, exactly, and a score of ln n
    rounded to fp32 leaves what the logarithm of n is off by."""
    V = 4096
    n = torch.arange(1, V + 1, device="cuda")
    x = torch.where(torch.arange(V, device="cuda") < n[:, None], 1.5, -math.inf)
    scores = torch.log(n.double()).float()
    s, t, _ = beam.select(x, scores[:, None].contiguous())
    want = scores.double() - torch.log(n.double())
    assert bool(((s[:, 0].double() - want).abs() <= 1.4e-9 + 2.0 ** -24 * want.abs()).all())
    assert (t == 0).all()
