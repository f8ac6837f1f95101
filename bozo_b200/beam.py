"""Beam search: the choice of the best continuations of several hypotheses a prompt.

``select`` is the operator; ``serving.beam_search`` is the search on paged caches, with
``paged.fork`` and ``paged.copy_pages`` reordering what the hypotheses hold.  The
reference only samples (model.py:718-768).
"""
from __future__ import annotations

from typing import Optional, Tuple

from torch import Tensor

from . import _capi

__all__ = ["select"]


def select(logits: Tensor, scores: Tensor, *, done: Optional[Tensor] = None,
           eos: Optional[int] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """The K best continuations of each prompt's K hypotheses.

    logits : ``[N · K, V]`` (fp32, bf16 or fp16; rows contiguous, any stride between
             them), row n·K + k that of prompt n's hypothesis k.
    scores : ``[N, K]`` float32, each hypothesis' sum of log probabilities; −∞ for one
             that does not take part (at the start all but the first of a prompt).
    done   : ``[N, K]`` bool, hypotheses that have ended: each goes on as itself only,
             with token ``eos`` and its score unchanged.

    A continuation is worth score + logit − log Σ exp(logits), added up and compared in 64
    bits; of equal ones the lower hypothesis comes first, of one hypothesis the higher logit,
    then the lower token.  The exponentials are summed from 32-bit ones: log Σ exp is off by
    a few 1e-7, and by (79 + 2.3 ln V) · 2^-24 at most, so continuations of two hypotheses
    closer than that may come in either order.  A masked token (logit −∞), and every token of a row with a NaN or
    +∞, of a row of −∞ only, or of a hypothesis whose score is not finite, is worth −∞:
    those come last, lowest token first.

    Returns ``scores [N, K]`` (float32, best first), ``tokens [N, K]`` (int64) and
    ``rows [N, K]`` (int32): the row of ``logits`` that each continues.  K up to 32, V
    from K to 2^20, N · K up to 65535.  No gradients."""
    return _capi.ext().beam_select(logits, scores, done, -1 if eos is None else int(eos))
