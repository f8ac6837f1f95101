"""Serving TensionLM: sequences that come and go, decoded together.

``decode`` decodes a batch in lock step — every sequence at one position, each
with rings of its own.  Here a batch has ``slots``, each idle or holding a
sequence at its own position, over the paged caches of ``bozo_b200.paged``:

* a local layer needs its last ``window`` tokens only: each slot has a ring of
  ⌈(W + 1) / page⌉ pages for good;
* global layers take pages of a shared pool as their sequences grow, and give
  them back when a sequence is released — one page table for all global layers
  (a page number stands for that page of every layer's pool).

``PagedState`` holds the caches; ``admit`` takes prompts of any lengths in one
forward, ``extend`` adds further tokens to a held sequence (the next turn of a
conversation), ``step`` feeds one token to every active slot, ``release`` frees
a slot.  ``PagedStepGraph`` replays the step as a CUDA graph: positions and page
tables are read on the device, so admitting, releasing and growing between
replays need no new capture.  ``generate`` is continuous batching on top: a
queue of prompts over the slots, ``decode.generate``'s sampling for each.

A step's logits equal those of ``decode.step`` for each sequence on its own, past
``max_seq_len`` tokens where the page size divides it: global layers reach whole
pages, so up to ``page_size − 1`` keys more otherwise.
The caches may be held in 8 bits (``cache_dtype`` e4m3 or int8), a quarter of
fp32 and half of bf16 plus 4 bytes a row.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch
from torch import Tensor

from . import _capi, decode, ops, paged

__all__ = ["PagedState", "PagedStepGraph", "admit", "extend", "step", "generate"]


class _Layer:
    """One layer's pages (and scales)."""

    def __init__(self, pages: int, heads: int, page: int, width: int, dtype: torch.dtype, dev):
        self.k, self.v = (torch.zeros(pages, heads, page, width, dtype=dtype, device=dev) for _ in "kv")
        eight = dtype in (torch.float8_e4m3fn, torch.int8)
        self.scales = {n: torch.zeros(pages, heads, page, device=dev) if eight else None
                       for n in ("k_scale", "v_scale")}


class PagedState:
    """Caches of up to ``slots`` sequences.

    max_len    : longest sequence (prompt and generated) the RoPE tables cover.
    page_size  : tokens of a page (multiples of 16 read fastest).
    pages      : pages of the global layers' pool (default: enough for every
                 slot at its longest).
    dtype      : dtype of the projections the model produces (default: its
                 parameters').
    cache_dtype: dtype of the pages (default: ``dtype``).

    A global layer reaches the last ``ceil(min(max_len, max_seq_len) /
    page_size)`` pages of its sequence.
    """

    def __init__(self, model, slots: int, max_len: int, *, page_size: int = 16,
                 pages: Optional[int] = None, dtype: Optional[torch.dtype] = None,
                 cache_dtype: Optional[torch.dtype] = None):
        cfg = model.cfg
        dev = next(model.parameters()).device
        if dev.type != "cuda":
            raise RuntimeError("serving runs on the CUDA decode kernels: move the model to a GPU")
        if slots < 1 or max_len < 1 or page_size < 1:
            raise ValueError("slots, max_len and page_size must be at least 1")
        if not cfg.use_rope and max_len > cfg.max_seq_len:
            raise ValueError("learned positions reach max_seq_len: max_len must not pass it")
        self.model, self.slots, self.max_len, self.page_size = model, slots, max_len, page_size
        self.dtype = dtype or next(model.parameters()).dtype
        cache_dtype = cache_dtype or self.dtype
        ring = -(-(cfg.window + 1) // page_size)
        reach = -(-min(max_len, cfg.max_seq_len) // page_size)
        pages = slots * reach if pages is None else pages
        self.local_table = torch.arange(slots * ring, dtype=torch.int32, device=dev).view(slots, ring)
        self.global_table = torch.full((slots, reach), -1, dtype=torch.int32, device=dev)
        self.layers = [_Layer(pages if b.global_layer else slots * ring, cfg.num_heads, page_size,
                              cfg.head_dim, cache_dtype, dev) for b in model.blocks]
        self.has_global = any(b.global_layer for b in model.blocks)
        self.lengths = torch.full((slots,), -1, dtype=torch.int32, device=dev)
        self.rope = ops.rope_tables(cfg.head_dim, max_len, 10_000.0, dev) if cfg.use_rope else None
        self._len: List[Optional[int]] = [None] * slots       # host copies: tokens held,
        self._pages: List[List[int]] = [[] for _ in range(slots)]  # global pages owned
        self._free = list(range(pages - 1, -1, -1))

    # ── host side: slots and pages ──

    @property
    def idle(self) -> List[int]:
        """Slots without a sequence."""
        return [i for i, n in enumerate(self._len) if n is None]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, slot: int) -> int:
        """Tokens the slot's sequence holds."""
        n = self._len[slot]
        if n is None:
            raise ValueError(f"slot {slot} is idle")
        return n

    def _grow(self, want) -> None:
        """Own pages for ``want = {slot: tokens}`` in all; nothing changes where
        they do not all fit."""
        if not self.has_global:
            return
        reach = self.global_table.shape[1]
        need = {s: min(reach, -(-n // self.page_size)) - len(self._pages[s]) for s, n in want.items()}
        need = {s: n for s, n in need.items() if n > 0}
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"out of pages: {sum(need.values())} wanted, {len(self._free)} free "
                               "(release a sequence, or give PagedState more pages)")
        rows, cols, new = [], [], []
        for s, n in need.items():
            for _ in range(n):
                rows.append(s)
                cols.append(len(self._pages[s]))
                new.append(self._free.pop())
                self._pages[s].append(new[-1])
        if new:
            at = torch.tensor([rows, cols, new]).to(self.lengths.device)
            self.global_table[at[0], at[1]] = at[2].int()

    def _check(self, tokens: int) -> None:
        if tokens > self.max_len:
            raise ValueError(f"a sequence of {tokens} tokens does not fit max_len {self.max_len}")

    def release(self, slot: int) -> None:
        """Give up a slot's sequence; its pages go back to the pool."""
        self.length(slot)
        self._free.extend(reversed(self._pages[slot]))
        self._pages[slot] = []
        self._len[slot] = None
        self.lengths[slot] = -1
        self.global_table[slot] = -1

    # ── device side ──

    def table(self, li: int) -> Tensor:
        return self.global_table if self.model.blocks[li].global_layer else self.local_table

    def _write(self, li: int, table: Tensor, start: Tensor, cu: Tensor, k: Tensor, v: Tensor) -> None:
        lay = self.layers[li]
        paged.write_kv(k, v, lay.k, lay.v, table, start, cu_rows=cu, rope=self.rope, **lay.scales)


@torch.no_grad()
def admit(state: PagedState, prompts: Sequence[Sequence[int]]):
    """Take ``prompts`` (lists of ids, any lengths up to ``max_seq_len``) into idle
    slots in one forward; returns (slots, logits ``[n, V]`` after each prompt)."""
    model, cfg = state.model, state.model.cfg
    lens = [len(p) for p in prompts]
    slots = state.idle[:len(prompts)]
    if not prompts or min(lens) < 1 or max(lens) > cfg.max_seq_len:
        raise ValueError(f"admit: prompts of 1 to {cfg.max_seq_len} ids are wanted")
    if len(slots) < len(prompts):
        raise RuntimeError(f"admit: {len(prompts)} prompts, {len(slots)} idle slots")
    for n in lens:
        state._check(n)
    state._grow(dict(zip(slots, lens)))
    dev, T = state.lengths.device, max(lens)
    ids = torch.tensor([list(p) + [0] * (T - n) for p, n in zip(prompts, lens)], device=dev)
    at = torch.tensor(slots, device=dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device=dev)
    cu[1:] = n.cumsum(0)
    start = torch.zeros_like(n)
    # the padded forward's rows that are tokens (its padding comes after them)
    rows = torch.cat([torch.arange(m) + i * T for i, m in enumerate(lens)]).to(dev)
    packed = len(rows) == ids.numel()
    x = model.embedding(ids)
    if model.pos_embedding is not None:
        x = x + model.pos_embedding(model.pos_buf[:, :T])
    for li, blk in enumerate(model.blocks):
        h = blk.pre_norm(x)
        _, k, v = blk.tension.project(h)
        k, v = (y.flatten(0, 1) if packed else y.flatten(0, 1)[rows] for y in (k, v))
        state._write(li, state.table(li)[at], start, cu, k, v)
        x = blk.ffn(blk._osc(blk.tension(h)))
    last = x[torch.arange(len(lens), device=dev), n.long() - 1]
    logits = model.lm_head(model.final_norm(last))
    state.lengths[at] = n
    for s, m in zip(slots, lens):
        state._len[s] = m
    return slots, logits


@torch.no_grad()
def extend(state: PagedState, slot: int, ids: Sequence[int]) -> Tensor:
    """Add ``ids`` to a held sequence in one forward over them; returns the logits
    ``[V]`` after the last.  The earlier keys and values that the new tokens
    reach are read back from the pages.  Tokens past a global layer's reach attend
    its last keys as they would in a step, one after another in those layers.
    Where it fails midway (out of memory), rings may hold some of the new rows:
    release the slot."""
    model, cfg = state.model, state.model.cfg
    t, T = state.length(slot), len(ids)
    if T < 1:
        raise ValueError("extend: at least one id is wanted")
    state._check(t + T)
    state._grow({slot: t + T})
    dev = state.lengths.device
    at = torch.tensor([slot], device=dev)
    x = model.embedding(torch.tensor([list(ids)], device=dev))
    pos = torch.arange(t, t + T, device=dev)
    at32 = pos.int()
    start = at32[:1]
    if model.pos_embedding is not None:
        x = x + model.pos_embedding(pos)
    for li, blk in enumerate(model.blocks):
        layer, lay, table = blk.tension, state.layers[li], state.table(li)[at]
        h = blk.pre_norm(x)
        q, k, v = layer.project(h)
        # tokens that reach all before them go together; past a global layer's last
        # pages each new row takes the place of the oldest that the one before reaches
        cap = table.shape[1] * state.page_size
        m = min(T, max(0, cap - t)) if layer.global_layer else T
        msg = [_chunk(state, li, table, start, t, q[:, :m], k[:, :m], v[:, :m])] if m else []
        for i in range(m, T):
            msg.append(paged.paged_tension(
                q[:, i], lay.k, lay.v, table, at32[i:i + 1], window=None, scale=layer.scale, rope=state.rope,
                k=k[:, i], v=v[:, i], **lay.scales).unsqueeze(1))
        msg = msg[0] if len(msg) == 1 else torch.cat(msg, dim=1)
        hh = layer.norm.wo_add_forward(h, msg.reshape(1, T, -1), layer.wo, layer.dropout)
        x = blk.ffn(_oscillate(blk, hh, pos[None, :, None]))
    state.lengths[slot] = t + T
    state._len[slot] = t + T
    return model.lm_head(model.final_norm(x[0, -1]))


def _chunk(state: PagedState, li: int, table: Tensor, start: Tensor, t: int, q: Tensor, k: Tensor,
           v: Tensor) -> Tensor:
    """One layer's tension ``[1, T, H, HD]`` of T new tokens from position t on that
    reach every key before them (of a local layer, in their window)."""
    cfg, layer, lay = state.model.cfg, state.model.blocks[li].tension, state.layers[li]
    T, dev = q.shape[1], q.device
    # the held rows that the first new query reaches come first, then the new
    # ones, written only now: a ring may put them in the old ones' place
    back = t if layer.global_layer else min(t, cfg.window)
    kk, vv = paged.read_kv(lay.k, lay.v, table, start - back, torch.tensor([0, back], dtype=torch.int32, device=dev),
                           back, dtype=k.dtype, **lay.scales)
    state._write(li, table, start, torch.tensor([0, T], dtype=torch.int32, device=dev), k[0], v[0])
    if state.rope is not None:
        q, k = (decode._rotate(y, state.rope[0], state.rope[1], t).to(y.dtype) for y in (q, k))
    kk = torch.cat([kk[None], k], dim=1)
    vv = torch.cat([vv[None], v], dim=1)
    qq = torch.cat([q.new_zeros(1, back, *q.shape[2:]), q], dim=1)
    return ops.tension(qq, kk, vv, window=None if layer.global_layer else cfg.window, scale=layer.scale,
                       rope_base=None, normalize="mass" if layer.global_layer else "count")[:, back:]


def _oscillate(blk, x: Tensor, pos: Tensor) -> Tensor:
    """model.py:303-310 at positions ``pos`` (broadcast against x's tokens)."""
    osc = blk.oscillate
    if osc is None:
        return x
    return x * (1.0 + osc.amp * torch.sin(pos.float() * osc.freqs + osc.phases))


def _check_tokens(state: PagedState, tokens: Tensor) -> None:
    if tokens.shape != (state.slots,):
        raise ValueError(f"step: tokens must be [{state.slots}], got {tuple(tokens.shape)}")
    if tokens.dtype == torch.bool or tokens.is_floating_point() or tokens.is_complex():
        raise TypeError(f"step: tokens must be integers, got {tokens.dtype}")


def _reserve(state: PagedState) -> dict:
    """Pages for a step's new tokens; the lengths after it, by slot."""
    held = {s: n + 1 for s, n in enumerate(state._len) if n is not None}
    for n in held.values():
        state._check(n)
    state._grow(held)
    return held


def _advance(state: PagedState, held: dict) -> None:
    """The step is under way: the host's lengths follow the device's."""
    for s, n in held.items():
        state._len[s] = n
    ops.check_device_error(state.lengths.device)


@torch.no_grad()
def _step(state: PagedState, tokens: Tensor, export: bool):
    """Device side of a step: reads device state only."""
    model, cfg = state.model, state.model.cfg
    D = cfg.dim
    x = model.embedding(tokens).unsqueeze(1)
    pos = state.lengths.clamp(min=0)
    if model.pos_embedding is not None:
        x = x + model.pos_embedding(pos.long()).unsqueeze(1)
    rows = []
    for li, blk in enumerate(model.blocks):
        layer, lay = blk.tension, state.layers[li]
        h = blk.pre_norm(x)
        q, k, v = layer.project(h)
        glob = layer.global_layer
        res = paged.paged_tension(
            q[:, 0], lay.k, lay.v, state.table(li), state.lengths, window=None if glob else cfg.window,
            scale=layer.scale, normalize="mass" if export or glob else "count", rope=state.rope,
            k=k[:, 0], v=v[:, 0], return_tau=export, tau_window=cfg.window if export else None,
            **lay.scales)
        out, tau = res if export else (res, None)
        hh = layer.norm.wo_add_forward(h, out.view(-1, 1, D), layer.wo, layer.dropout)
        x = blk.ffn(_oscillate(blk, hh, pos[:, None, None]))
        rows.append(tau)
    logits = model.lm_head(model.final_norm(x))[:, 0]
    state.lengths += (state.lengths >= 0).int()
    return (logits, rows) if export else logits


def step(state: PagedState, tokens: Tensor, export: bool = False):
    """Feed one token to every active slot (``tokens [slots]``; idle slots' entries
    are ignored); returns the logits ``[slots, V]`` and with ``export`` each
    layer's τ rows ``[slots, H, W]`` (as ``decode.step``, zeros in idle slots)."""
    _check_tokens(state, tokens)
    if tokens.device != state.lengths.device:
        raise ValueError(f"step: tokens must be on {state.lengths.device}, got {tokens.device}")
    held = _reserve(state)
    res = _step(state, tokens.long(), export)
    _advance(state, held)
    return res


class PagedStepGraph:
    """``step(state, tokens, export)`` captured as one CUDA graph.  Sequences may
    be admitted, extended and released between calls; the returned tensors are
    the graph's buffers, overwritten by the next call."""

    def __init__(self, state: PagedState, export: bool = False, warmup: int = 2):
        self.state = state
        dev = state.lengths.device
        self.tokens = torch.zeros(state.slots, dtype=torch.long, device=dev)
        held = state.lengths.clone()
        side = torch.cuda.Stream(dev)
        try:
            state.lengths.fill_(-1)  # every slot idle: nothing is written
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                for _ in range(warmup):
                    _step(state, self.tokens, export)
            torch.cuda.current_stream(dev).wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = _step(state, self.tokens, export)
        finally:
            torch.cuda.current_stream(dev).wait_stream(side)
            state.lengths.copy_(held)

    def __call__(self, tokens: Tensor):
        _check_tokens(self.state, tokens)
        self.tokens.copy_(tokens)
        held = _reserve(self.state)
        self.graph.replay()
        _advance(self.state, held)
        return self.out


@torch.no_grad()
def generate(model, prompts: Sequence[Sequence[int]], max_new: int = 200, temp: float = 0.8,
             top_p: float = 0.92, rep_penalty: float = 1.3, slots: int = 16,
             dtype: Optional[torch.dtype] = None, cache_dtype: Optional[torch.dtype] = None,
             page_size: int = 16, graph: bool = True) -> List[List[int]]:
    """``decode.generate`` for many prompts: up to ``slots`` sequences at a time,
    the next prompts admitted as others end.  Returns each prompt followed by
    its new ids."""
    model.eval()
    out = [list(p) for p in prompts]
    limit = model.cfg.max_seq_len
    # the last max_seq_len ids are the context; without RoPE PagedState refuses what
    # would pass them
    ctx = [p[-limit:] for p in out]
    queue = list(range(len(ctx))) if max_new > 0 else []
    if not queue:
        return out
    longest = max(len(ctx[i]) for i in queue) + max_new
    slots = min(slots, len(queue))
    state = PagedState(model, slots, longest, page_size=page_size, dtype=dtype, cache_dtype=cache_dtype)
    dev = state.lengths.device
    run = PagedStepGraph(state) if graph else (lambda tok: step(state, tok))
    who: dict = {}                       # slot → prompt
    left = [max_new] * len(out)
    pending: dict = {}                   # slot → token to feed

    def take(slot: int, logits: Tensor) -> None:
        i = who[slot]
        nxt = decode._sample(logits, out[i][-32:], temp, top_p, rep_penalty)
        out[i].append(nxt)
        left[i] -= 1
        if left[i]:
            pending[slot] = nxt
        else:
            pending.pop(slot, None)
            state.release(slot)
            del who[slot]

    while queue or pending:
        n = min(len(queue), len(state.idle))
        if n:
            batch, queue = queue[:n], queue[n:]
            got, logits = admit(state, [ctx[i] for i in batch])
            who.update(zip(got, batch))
            for slot, row in zip(got, logits):
                take(slot, row)
            continue
        tok = torch.tensor([pending.get(s, 0) for s in range(slots)], device=dev)
        logits = run(tok).clone()
        for slot in list(pending):
            take(slot, logits[slot])
    return out
