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
``beam_search`` keeps several hypotheses of each prompt (``BeamState``): a step
takes their pages, feeds their tokens, chooses the best continuations and
reorders tables and caches on the device, in one CUDA graph a token.

A step's logits equal those of ``decode.step`` for each sequence on its own, past
``max_seq_len`` tokens where the page size divides it: global layers reach whole
pages, so up to ``page_size − 1`` keys more otherwise.
The caches may be held in 8 bits (``cache_dtype`` e4m3 or int8), a quarter of
fp32 and half of bf16 plus 4 bytes a row, or in 4 (``torch.float4_e2m1fn_x2``), half
of that plus a byte for 16 elements.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _capi, beam, decode, ops, paged

__all__ = ["PagedState", "PagedStepGraph", "BeamState", "admit", "extend", "step", "generate", "beam_search"]


class _Layer:
    """One layer's pages (and scales)."""

    def __init__(self, pages: int, heads: int, page: int, width: int, dtype: torch.dtype, dev):
        four = dtype == torch.float4_e2m1fn_x2
        shape = (pages, heads, page, width // 2 if four else width)
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8 if four else dtype, device=dev) for _ in "kv")
        scaled = four or dtype in (torch.float8_e4m3fn, torch.int8)
        self.scales = {n: torch.zeros(pages, heads, page, device=dev) if scaled else None
                       for n in ("k_scale", "v_scale")}
        if four:
            self.k, self.v = self.k.view(dtype), self.v.view(dtype)
            self.scales.update({n: torch.zeros(pages, heads, page, width // 16, dtype=torch.float8_e4m3fn, device=dev)
                                for n in ("k_group", "v_group")})

    @property
    def pools(self) -> List[Tensor]:
        """Everything that is held by pages."""
        return [self.k, self.v] + [s for s in self.scales.values() if s is not None]


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
        if cache_dtype == torch.float4_e2m1fn_x2 and cfg.head_dim % 16:
            raise ValueError("4-bit caches hold heads of a multiple of 16 elements")
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

    @property
    def tables(self) -> dict:
        """The page tables: of the global layers (``True``) and of the local ones."""
        return {True: self.global_table, False: self.local_table}

    def table(self, li: int) -> Tensor:
        return self.tables[bool(self.model.blocks[li].global_layer)]

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
    logits = _prefill(state, ids, n.long(), rows, {g: t[at] for g, t in state.tables.items()}, start, cu)
    state.lengths[at] = n
    for s, m in zip(slots, lens):
        state._len[s] = m
    return slots, logits


def _prefill(state: PagedState, ids: Tensor, n: Tensor, rows: Tensor, tables: dict, start: Tensor,
             cu: Tensor) -> Tensor:
    """The model over padded prompts ``ids [B, T]`` of ``n [B]`` tokens, whose packed rows
    are ``rows`` of the flattened batch: their keys and values into the caches, the
    logits ``[B, V]`` after each."""
    model, T = state.model, ids.shape[1]
    packed = len(rows) == ids.numel()
    x = model.embedding(ids)
    if model.pos_embedding is not None:
        x = x + model.pos_embedding(model.pos_buf[:, :T])
    for li, blk in enumerate(model.blocks):
        h = blk.pre_norm(x)
        _, k, v = blk.tension.project(h)
        k, v = (y.flatten(0, 1) if packed else y.flatten(0, 1)[rows] for y in (k, v))
        state._write(li, tables[bool(blk.global_layer)], start, cu, k, v)
        x = blk.ffn(blk._osc(blk.tension(h)))
    last = x[torch.arange(len(ids), device=ids.device), n - 1]
    return model.lm_head(model.final_norm(last))


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
        state._grow({})  # refused by states that are not fed slot by slot
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


class BeamState(PagedState):
    """``beams`` hypotheses of each of up to ``prompts`` prompts, searched together on the
    device: hypothesis k of prompt n has slot n · beams + k.

    The pages of both kinds of layers are counted on the device (``paged.reserve``,
    ``paged.fork``): hypotheses share the full pages of what they have in common, and
    the rings of local layers move or are copied with them.  ``start`` takes the
    prompts, ``advance`` adds a token to every hypothesis (a replayed CUDA graph unless
    ``graph=False``), ``results`` reads what was found.  The calls for single slots
    (``admit``, ``extend``, ``step``, ``PagedStepGraph``, ``release`` and the like) are
    refused.

    max_len : longest prompt with its new tokens; with global layers at most
              ``max_seq_len``, since shared pages cannot be rings.
    eos     : token that ends a hypothesis, or ``None``.
    """

    def __init__(self, model, prompts: int, beams: int, max_len: int, *, eos: Optional[int] = None,
                 page_size: int = 16, dtype: Optional[torch.dtype] = None,
                 cache_dtype: Optional[torch.dtype] = None, graph: bool = True, warmup: int = 2):
        cfg = model.cfg
        if prompts < 1 or not 1 <= beams <= 32 or beams > cfg.vocab_size:
            raise ValueError("beam search takes at least one prompt and 1 to 32 beams, no more than tokens")
        if prompts * beams > 8192:
            raise ValueError(f"beam search holds up to 8192 hypotheses, not {prompts} prompts of {beams}")
        if eos is not None and not 0 <= eos < cfg.vocab_size:
            raise ValueError(f"eos must be a token, got {eos}")
        if any(b.global_layer for b in model.blocks) and max_len > cfg.max_seq_len:
            raise ValueError(f"beam search holds whole sequences: {max_len} tokens pass max_seq_len {cfg.max_seq_len}")
        super().__init__(model, prompts * beams, max_len, page_size=page_size, dtype=dtype, cache_dtype=cache_dtype)
        dev = self.lengths.device
        self.prompts, self.beams, self.eos = prompts, beams, eos
        # by kind of layer (global or not): what its pages hold, and how many rows hold a page
        self.pools = {g: [p for lay, b in zip(self.layers, model.blocks) if bool(b.global_layer) == g
                          for p in lay.pools] for g in sorted({bool(b.global_layer) for b in model.blocks})}
        self.refs = {g: torch.zeros(p[0].shape[0], dtype=torch.int32, device=dev) for g, p in self.pools.items()}
        self.local_table.fill_(-1)  # pages of rings, too, go from hypothesis to hypothesis
        self.tokens = torch.zeros(self.slots, dtype=torch.long, device=dev)
        self.scores = torch.zeros(prompts, beams, device=dev)
        self.done = None if eos is None else torch.zeros(prompts, beams, dtype=torch.bool, device=dev)
        # what each step chose: tokens, and the slots that were continued
        self.chosen = torch.zeros(max_len, 2, self.slots, dtype=torch.long, device=dev)
        self.steps = torch.zeros(1, dtype=torch.long, device=dev)
        self.taken = 0
        self._graph = None
        if graph:
            # nothing is held yet: every slot is idle, and no page moves
            side = torch.cuda.Stream(dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                for _ in range(warmup):
                    self._advance()
                    self.steps.zero_()
            torch.cuda.current_stream(dev).wait_stream(side)
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                self._advance()
            self._graph = captured

    # What counts slots and pages on the host (admit, extend, step, PagedStepGraph, release)
    # knows nothing of the device's counts.

    def _together(self, *_) -> None:
        raise RuntimeError("a beam search's slots are taken, fed and given up together: start() takes new "
                           "prompts, advance() adds a token to all")

    length = release = _grow = _together
    idle = free_pages = property(_together)

    @torch.no_grad()
    def start(self, prompts: Sequence[Sequence[int]]) -> None:
        """Take new prompts (lists of ids of 1 to ``max_seq_len``, as many as there is room
        for); what was held before is given up."""
        K, dev = self.beams, self.lengths.device
        lens = [len(p) for p in prompts]
        if len(prompts) != self.prompts or min(lens) < 1 or max(lens) > min(self.max_len, self.model.cfg.max_seq_len):
            raise ValueError(f"start: {self.prompts} prompts of 1 to {min(self.max_len, self.model.cfg.max_seq_len)} "
                             "ids are wanted")
        T = max(lens)
        ids = torch.tensor([list(p) + [0] * (T - m) for p, m in zip(prompts, lens)], device=dev)
        n = torch.tensor(lens, device=dev)
        self.taken = 0  # a call that fails from here on leaves nothing to advance
        for g in self.pools:
            self.tables[g].fill_(-1)
            self.refs[g].zero_()
        self.lengths.fill_(-1)
        self.lengths[::K] = 0
        tokens = torch.zeros(self.slots, dtype=torch.int32, device=dev)
        tokens[::K] = n.int()
        for g in self.pools:
            plan = self._reserve(g, tokens, rows=sum(lens))
        rows = plan.seq.long() // K * T + plan.pos  # of the padded batch
        logits = _prefill(self, ids, n, rows, self.tables, self.lengths, plan.cu_rows)
        self.lengths[::K] = n.int()
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0
        if self.done is not None:
            self.done.zero_()
        self.steps.zero_()
        self.longest = T
        self._choose(logits.repeat_interleave(K, 0))
        self.taken = 1

    def _started(self) -> None:
        if not self.taken:
            raise RuntimeError("nothing is searched: start() takes the prompts first")

    def advance(self) -> None:
        """Feed every hypothesis its token and choose the best continuations."""
        self._started()
        self._check(self.longest + self.taken)
        taken, self.taken = self.taken, 0  # as in start()
        if self._graph is not None:
            self._graph.replay()
        else:
            self._advance()
        self.taken = taken + 1
        ops.check_device_error(self.lengths.device)

    def _reserve(self, glob: bool, tokens: Optional[Tensor], rows: Optional[int] = None) -> paged.Plan:
        return paged.reserve(self.tables[glob], self.lengths, tokens, self.refs[glob], self.page_size, rows=rows)

    @torch.no_grad()
    def _advance(self) -> None:
        for g in self.pools:
            self._reserve(g, None)
        self._choose(_step(self, self.tokens, False))

    def _choose(self, logits: Tensor) -> None:
        scores, tokens, rows = beam.select(logits, self.scores, done=self.done, eos=self.eos)
        rows = rows.view(-1)
        for g, pools in self.pools.items():
            # none is missing: both pools have a page for every entry of their table
            copies, _ = paged.fork(self.tables[g], self.lengths, rows, self.refs[g], self.page_size, share=g)
            paged.copy_pages(pools, copies)
        at = rows.long()
        self.lengths.copy_(self.lengths[at])
        self.scores.copy_(scores)
        if self.done is not None:
            self.done.copy_(self.done.view(-1)[at].view_as(scores) | (tokens == self.eos))
        self.tokens.copy_(tokens.view(-1))
        self.chosen.index_copy_(0, self.steps, torch.stack([self.tokens, at]).unsqueeze(0))
        self.steps += 1

    def results(self, length_penalty: float = 0.0) -> List[List[Tuple[List[int], float]]]:
        """For each prompt its hypotheses' new ids (up to and with ``eos``) and scores, each
        the sum of log probabilities over (number of new ids) ^ ``length_penalty``, best
        first."""
        self._started()
        tokens, rows = self.chosen[:self.taken].cpu().unbind(1)
        scores, out = self.scores.tolist(), []
        for n in range(self.prompts):
            found = []
            for k in range(self.beams):
                r, ids = n * self.beams + k, []
                for t in range(self.taken - 1, -1, -1):
                    ids.append(int(tokens[t, r]))
                    r = int(rows[t, r])
                ids.reverse()
                if self.eos in ids:
                    ids = ids[:ids.index(self.eos) + 1]
                found.append((ids, scores[n][k] / len(ids) ** length_penalty))
            out.append(sorted(found, key=lambda x: -x[1]))
        return out


def beam_search(model, prompts: Sequence[Sequence[int]], beams: int = 4, max_new: int = 64, *,
                eos: Optional[int] = None, length_penalty: float = 0.0, batch: int = 16,
                dtype: Optional[torch.dtype] = None, cache_dtype: Optional[torch.dtype] = None,
                page_size: int = 16, graph: bool = True) -> List[List[Tuple[List[int], float]]]:
    """The ``beams`` best continuations of each prompt by beam search, ``batch`` prompts at
    a time: for each prompt ``(new ids, score)``, best first, as ``BeamState.results``
    returns them.  Longer prompts keep their last ``max_seq_len`` ids, or their last
    ``max_seq_len − max_new + 1`` where the model has global layers or learned positions."""
    model.eval()
    if max_new < 1 or batch < 1:
        raise ValueError("max_new and batch must be at least 1")
    cfg, out = model.cfg, []
    bounded = not cfg.use_rope or any(b.global_layer for b in model.blocks)
    limit = cfg.max_seq_len - max_new + 1 if bounded else cfg.max_seq_len
    if limit < 1:
        raise ValueError(f"{max_new} new tokens do not fit max_seq_len {cfg.max_seq_len}")
    ctx = [list(p)[-limit:] for p in prompts]
    for i in range(0, len(ctx), batch):
        part = ctx[i:i + batch]
        state = BeamState(model, len(part), beams, max(map(len, part)) + max_new - 1, eos=eos,
                          page_size=page_size, dtype=dtype, cache_dtype=cache_dtype, graph=graph and max_new > 1)
        state.start(part)
        for step_ in range(1, max_new):
            # the host looks at the ended hypotheses now and then
            if eos is not None and step_ % 8 == 0 and bool(state.done.all()):
                break
            state.advance()
        ops.poll_device_error(state.lengths.device)
        out += state.results(length_penalty)
    return out
