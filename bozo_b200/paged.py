"""Paged key/value caches: sequences of different lengths, each at its own
position, in pages of a shared pool — in fp32, bf16 or fp16, or in 8 bits
(e4m3 or integers) with one fp32 scale a row, or in 4 bits (e2m1) with one e4m3
scale for 16 elements besides.

The reference keeps no keys between tokens (model.py:718-768 re-runs the whole
context for each one) and ``decode.DecodeState`` keeps rings for a batch that
decodes in lock step; these are the operators for a batch whose sequences come
and go:

* ``write_kv``: rotates new tokens' keys, and writes (quantises) their keys and
  values into the pages — whole prompts of ragged lengths or one token each;
* ``read_kv``: reads rows back, dequantised;
* ``paged_tension``: the tension of one new token a sequence over its cached
  keys (with the new token's key and value written first when they are given).

and for the page tables, kept on the device:

* ``reserve``: pages for new tokens, and where each of them goes;
* ``fork``: rows of the table reordered, dropped and multiplied (the hypotheses of
  a beam search), with the pages that have to be copied for it;
* ``copy_pages``: those copies, in every layer's pools.

The first three take the same cache arguments:

* ``k_pages``, ``v_pages`` ``[P, Hk, page, HD]``, and ``k_scale``, ``v_scale``
  ``[P, Hk, page]`` (float32) for 8-bit pages;
* 4-bit pages are ``torch.float4_e2m1fn_x2`` ``[P, Hk, page, HD/2]`` (two elements a
  byte, the first in the low bits; HD a multiple of 16) and take ``k_group``,
  ``v_group`` ``[P, Hk, page, HD/16]`` (``torch.float8_e4m3fn``) as well: an element
  stands for (code · group) · scale;
* ``page_table [B, M]`` (int32): position s of sequence b lies in page
  ``page_table[b, (s mod C) // page]``, row ``s mod page``, with C = M·page: a
  table narrower than its sequence is a ring that keeps the last C tokens;
* ``lengths [B]`` (int32): the position of each sequence's (first) new token;
  negative for an inactive one, which is skipped and comes out as zeros.

Everything else is read on the device, so the calls can be captured in a CUDA
graph.  They run on the current stream of the pages' device; a position beyond
the RoPE tables or a page outside the pool is skipped and reported by
``check_device_error`` / ``poll_device_error``.  No gradients.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _capi, ops

__all__ = ["write_kv", "read_kv", "paged_tension", "Plan", "reserve", "fork", "copy_pages"]


def write_kv(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
             lengths: Tensor, *, cu_rows: Optional[Tensor] = None, rope=None,
             k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None,
             k_group: Optional[Tensor] = None, v_group: Optional[Tensor] = None) -> None:
    """Write new tokens' keys and values into the pages, in place.

    k, v    : ``[N, Hk, HD]`` pre-RoPE projections (any strides).
    cu_rows : ``[B + 1]`` int32 row offsets: sequence b's tokens are the rows
              ``cu_rows[b]:cu_rows[b+1]``, at positions ``lengths[b]``, …; rows
              before ``cu_rows[0]`` and from ``cu_rows[B]`` on are padding.
              ``None``: one row a sequence.
    rope    : ``(cos, sin, ...)`` tables ``[length, HD/2]`` (``ops.rope_tables``)
              for the keys, or ``None``.

    ``lengths`` is not advanced (all layers of a step share it).  Of more than C
    tokens of one sequence the last C are kept.
    """
    cos, sin = (rope[0], rope[1]) if rope is not None else (None, None)
    _capi.ext().paged_write(k, v, k_pages, v_pages, page_table, lengths, cu_rows, cos, sin,
                            k_scale, v_scale, k_group, v_group)


def read_kv(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, start: Tensor,
            cu_rows: Optional[Tensor], rows: int, *, k_scale: Optional[Tensor] = None,
            v_scale: Optional[Tensor] = None, k_group: Optional[Tensor] = None,
            v_group: Optional[Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    """Keys (rotated, as held) and values of ``rows`` cached tokens, each
    ``[rows, Hk, HD]`` in ``dtype``: rows ``cu_rows[b]:cu_rows[b+1]`` are sequence
    b's positions ``start[b]``, …; padding rows and inactive sequences are zeros.
    8-bit rows come back as code · scale, 4-bit ones as (code · group) · scale."""
    return _capi.ext().paged_read(k_pages, v_pages, page_table, start, cu_rows, rows, k_scale,
                                  v_scale, ops._dt(dtype), k_group, v_group)


def paged_tension(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                  lengths: Tensor, *, window: Optional[int], scale: Optional[float] = None,
                  normalize: Optional[str] = "mass", rope=None, k: Optional[Tensor] = None,
                  v: Optional[Tensor] = None, k_scale: Optional[Tensor] = None,
                  v_scale: Optional[Tensor] = None, k_group: Optional[Tensor] = None,
                  v_group: Optional[Tensor] = None, return_tau: bool = False,
                  tau_window: Optional[int] = None):
    """Tension of one new token a sequence, at position t = ``lengths[b]``.

    q        : ``[B, H, HD]`` pre-RoPE queries (any strides); H a multiple of Hk,
               query head h reads key head ``h // (H // Hk)``.
    window   : local look-back W (keys t − W … t − 1), or ``None`` for the global
               layer (keys up to and with t; the last C of them).
    scale    : dot divisor, default √HD.
    normalize: "mass", "count" (local only) or ``None`` / "none" (raw Σ τ·v).
    rope     : tables for q (and k), or ``None``.
    k, v     : ``[B, Hk, HD]`` the new token's projections, written first as
               ``write_kv`` does; without them a global layer expects them in the
               cache already.
    return_tau : also return the token's τ row ``[B, H, W]``: slot w is key
               t − (W − w) (local); ``[B, H, tau_window]``, column c is key t − c
               (global); zero where there is no key, or its page is outside the pool.

    Returns ``out [B, H, HD]`` in q's dtype, or ``(out, tau)``.  A NaN in a query or in
    a key that it reaches makes that query's output NaN, a NaN in a value that column
    of it; 8- and 4-bit rows with a NaN or an infinity are NaN as a whole.  An infinity in a
    16- or 32-bit value makes its column an infinity or NaN; one in a query or a key
    gives τ 0 or 1, or NaN, depending on the pages' type.  Neither reaches another
    sequence, another key head or, from a query, another query, and rows out of reach
    may hold anything.
    """
    norm = ops._NORM.get(normalize, -1)
    if norm < 0:
        raise ValueError(f"normalize must be 'mass', 'count' or None, got {normalize!r}")
    if window is None:
        mode, win, tw = _capi.MODE_GLOBAL, 0, int(tau_window or 0) if return_tau else 0
        if norm == _capi.NORM_COUNT:
            raise ValueError("normalize='count' is defined for local windows only")
        if return_tau and tw < 1:
            raise ValueError("global mode exports τ over the model's local window: pass tau_window")
    else:
        mode, win = _capi.MODE_LOCAL, int(window)
        tw = win if return_tau else 0
        if win < 1:
            raise ValueError("window must be >= 1")
        if return_tau and tau_window is not None and int(tau_window) != win:
            raise ValueError("a local window exports its own τ row: tau_window must be the window")
    cos, sin = (rope[0], rope[1]) if rope is not None else (None, None)
    return _capi.ext().paged_decode(q, k_pages, v_pages, page_table, lengths, mode, win, norm, scale,
                                    cos, sin, k, v, k_scale, v_scale, tw, k_group, v_group)


class Plan(NamedTuple):
    """What ``reserve`` returns, int32 on the device."""
    cu_rows: Tensor           # [B + 1]: new tokens before each sequence's
    missing: Tensor           # [1]: pages that were wanted and not there (then none was given)
    seq: Optional[Tensor]     # [rows]: a packed new token's sequence,
    pos: Optional[Tensor]     # its position,
    slot: Optional[Tensor]    # and its slot, page · page_size + row of the page; −1 without one


def reserve(page_table: Tensor, lengths: Tensor, tokens: Optional[Tensor], refs: Tensor,
            page_size: int, *, rows: Optional[int] = None) -> Plan:
    """Give every sequence's row of the page table the pages that its new tokens need.

    page_table : ``[B, M]`` int32, updated in place; entries outside the pool are empty.
    lengths    : ``[B]`` int32, tokens held; negative: an idle row, which gets none.
    tokens     : ``[B]`` int32, new tokens of each, or ``None``: one each.  Up to
                 2^31 / B of a sequence.
    refs       : ``[P]`` int32, how many rows hold each page of the pool (0: free);
                 updated in place.
    rows       : also say where the first ``rows`` packed new tokens go (``seq``, ``pos``,
                 ``slot``; −1 behind the last).  A token whose place a later one of this
                 call takes (a ring) has slot −1, one past position 2^31 − 1 has neither
                 (and is reported as an index error).

    Columns from ⌈lengths / page_size⌉ on are filled from the first empty one, up to
    ⌈(lengths + tokens) / page_size⌉ and M, so pages reserved before are kept.  Free
    pages are given in ascending order, to the sequences in theirs; where there are too
    few, no table row changes.  ``lengths`` is not advanced.  Up to 8192 sequences."""
    if rows is not None and rows < 0:
        raise ValueError("reserve: rows must not be negative")
    return Plan._make(_capi.ext().paged_reserve(page_table, lengths, tokens, refs, page_size,
                                                -1 if rows is None else rows))


def fork(page_table: Tensor, lengths: Tensor, parents: Tensor, refs: Tensor, page_size: int, *,
         share: bool = True) -> Tuple[Tensor, Tensor]:
    """Reorder the rows of a page table: row r becomes what row ``parents[r]`` was, −1
    empties it.  Pages that no row holds any more are free.

    page_table, refs : as in ``reserve``, both updated in place.
    lengths          : ``[B]`` int32, tokens held by the old rows (not changed: the caller
                       moves them along, ``lengths[parents]``).
    share            : full pages are held by all children of a row; the page being filled
                       stays with the first child, and each further one gets a free page
                       for a copy.  The table has to hold whole sequences (a row of more
                       than M · page_size tokens is reported as an index error).
                       ``False``: for rings, whose pages are all written again — the first
                       child keeps them, each further one gets copies of those in use.

    Returns ``copies`` (int32, ``[B, 2]`` or ``[B · M, 2]``: page to copy and its copy, −1
    where there is none) for ``copy_pages``, and ``missing [1]``: pages that were not there
    (the last rows then lack theirs; never where the pool has a page for every entry of the
    table, though where rows share pages a fork may want more than it gives up).  Free pages
    are given in ascending order."""
    return _capi.ext().paged_fork(page_table, lengths, parents, refs, page_size, share)


def copy_pages(pools: Sequence[Tensor], copies: Tensor) -> None:
    """Copy page ``copies[i, 0]`` to page ``copies[i, 1]`` in each of ``pools`` (contiguous
    ``[P, …]`` tensors of any type: pages, scales), skipping pairs outside the pool.  No
    page may be both read and written in one call, nor written twice."""
    _capi.ext().paged_copy(list(pools), copies)
