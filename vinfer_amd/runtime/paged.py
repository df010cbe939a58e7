"""The keys and values of a decode model in pages, its prompts shared: what ``BatchDecoder`` and ``beam_search`` need of
an attention model's state, over the ``paged`` operators. The engine's pool keeps one contiguous cache a slot
(src/vinfer/state/pool.py:41-128).

Request r's prompt is held once, in pages that are taken when it is prefilled; each of its beams (slots
``r * beams .. r * beams + beams - 1``) has the continuation to itself, in pages of its own that lie one after the other.
A step attends to both: the prompt's keys are read once for all beams. A search that changes beams moves the
continuations alone (``beam_states``), and a request's beams start without a copy of anything (``shared_prompts``).

    cache = SharedPromptCache(PAGED.resolve("hip", ctx), layers=.., requests=.., beams=.., ...)

    class Model:
        shared_prompts = True
        max_new_tokens = property(lambda self: cache.max_tokens)
        def prefill(self, slot, prompt_ids): step = cache.prefill(slot, len(prompt_ids)); ... step.attend(layer, q, k, v)
        def decode(self, slots, tokens, positions): step = cache.decode(slots, positions); ... step.attend(layer, q, k, v)
        def release(self, slot): cache.release(slot)
        def beam_states(self, slots): return cache.beam_states()

A decode step makes no host decision on what the device holds, so it can be captured into a graph.
"""

from __future__ import annotations

import torch

from vinfer_amd import _vpaged
from vinfer_amd.paged import AttentionPlan, PagedBackend, PageTables, Rotary
from vinfer_amd.runtime.batch import NoRoom
from vinfer_amd.sampler.beams import BeamState


class CacheStep:
    """One step's tokens: their positions and slots, and the attention's plan, for all layers."""

    def __init__(self, cache: SharedPromptCache, positions, slots, plan: AttentionPlan, tables, prefix_tables) -> None:
        self.cache, self.positions, self.slots, self.plan = cache, positions, slots, plan
        self.tables, self.prefix_tables = tables, prefix_tables

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Layer's attention ``[N, heads, head_dim]`` of the step's N tokens, whose keys and values are stored first;
        ``q`` and ``k`` as the projections gave them (they are turned here)."""
        c = self.cache
        q = c.backend.rotate_store(q, k, v, self.positions, self.slots, c.keys[layer], c.values[layer], c.rotary)
        out = c.backend.attend(q.view(self.plan.sequences, self.plan.queries, *q.shape[1:]), c.keys[layer], c.values[layer],
                               self.tables, self.plan, prefix_tables=self.prefix_tables, scale=c.scale)
        return out.view(q.shape)


class SharedPromptCache:
    """``requests`` prompts in ``prompt_pages`` pages together (each of up to ``max_prompt`` positions, 65536 at most), and
    ``max_tokens`` positions for each of their ``beams`` continuations."""

    def __init__(self, backend: PagedBackend, *, layers: int, requests: int, beams: int, heads: int, kv_heads: int, head_dim: int,
                 prompt_pages: int, max_prompt: int, max_tokens: int, rotary: Rotary, page_size: int = 16, dtype=torch.bfloat16,
                 device="cuda", scale: float | None = None) -> None:
        if min(layers, requests, beams, prompt_pages, max_prompt, max_tokens) < 1:
            raise ValueError("layers, requests, beams, prompt_pages, max_prompt and max_tokens must be positive")
        if max_prompt > _vpaged.MAX_QUERIES:  # (a prompt is one step's new tokens)
            raise ValueError(f"max_prompt must be at most {_vpaged.MAX_QUERIES}, got {max_prompt}")
        self.backend, self.rotary, self.scale = backend, rotary, scale
        self.requests, self.beams, self.max_prompt, self.max_tokens = requests, beams, max_prompt, max_tokens
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.layers, self.prompt_pages = layers, prompt_pages
        slots, own = requests * beams, -(-max_tokens // page_size)
        shape = layers, prompt_pages + slots * own, page_size, kv_heads, head_dim
        self.keys, self.values = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        dev = self.device = self.keys.device
        self.prompts = PageTables.empty(requests, -(-max_prompt // page_size), prompt_pages, page_size, dev)
        # a continuation's pages are its own from the start, one after the other: what reorders states can move them
        self.own_tables = (prompt_pages + torch.arange(slots * own, dtype=torch.int32, device=dev)).view(slots, own)
        self._starts = torch.arange(0, slots + 1, beams, dtype=torch.int32, device=dev)
        self._single = torch.arange(slots + 1, dtype=torch.int32, device=dev)

    def _one(self, request: int, n: int) -> torch.Tensor:
        t = torch.zeros(self.requests, dtype=torch.int32, device=self.device)
        t[request] = n
        return t

    def release(self, slot: int) -> None:
        """Give the pages of the prompt of ``slot``'s request back."""
        left = torch.full((self.requests,), (1 << 31) - 1, dtype=torch.int32, device=self.device)
        left[self._request(slot)] = 0
        self.backend.shrink(self.prompts, left)

    def _request(self, slot: int) -> int:
        if not 0 <= slot < self.requests * self.beams:
            raise ValueError(f"slot must be in [0, {self.requests * self.beams}), got {slot}")
        return slot // self.beams

    def prefill(self, slot: int, tokens: int) -> CacheStep:
        """The step of a prompt of ``tokens`` tokens, which takes the place of the one that ``slot``'s request had.
        ``NoRoom`` (a ``RuntimeError``) if there are too few pages left. Nothing is held for the request where this raises."""
        request = self._request(slot)
        if not 1 <= tokens <= self.max_prompt:
            raise ValueError(f"a prompt must have 1 to {self.max_prompt} tokens, got {tokens}")
        self.release(slot)
        e = self.backend.extend(self.prompts, self._one(request, tokens), tokens)
        if not bool(e.served[request]):
            raise NoRoom(f"no pages for a prompt of {tokens} tokens: {int(self.prompts.free_count)} are free")
        lengths, tables = self.prompts.lengths[request : request + 1], self.prompts.tables[request : request + 1]
        try:
            plan = self._plan(lengths, tokens, tables)
        except BaseException:
            self.release(slot)
            raise
        return CacheStep(self, e.positions, e.slots, plan, tables, None)

    def decode(self, slots: torch.Tensor, positions: torch.Tensor) -> CacheStep:
        """The step of one token at ``positions`` (in its prompt and continuation) for each of ``slots``: of a cache of
        several beams all of its slots in their order, of one beam any slots, each once. A token past its continuation's
        ``max_tokens`` places is none (only the device knows): nothing is stored and its attention is 0."""
        n = slots.shape[0]
        if self.beams > 1 and n != self.requests * self.beams:
            raise ValueError(f"a step of beams takes all {self.requests * self.beams} slots, got {n}")
        request = slots // self.beams if self.beams > 1 else slots
        prefix = self.prompts.lengths.index_select(0, request)
        own = positions.int() - prefix  # the token's place in its continuation
        tables = self.own_tables if self.beams > 1 else self.own_tables.index_select(0, slots)
        inside = (own >= 0) & (own < self.max_tokens)
        page = tables.gather(1, (own.clamp(0, self.max_tokens - 1) // self.page_size).long()[:, None])[:, 0]
        at = torch.where(inside, page * self.page_size + own % self.page_size, -1)
        lengths = torch.where(inside, own + 1, 0)
        if self.beams > 1:
            prefixes, prefix_tables, starts = self.prompts.lengths, self.prompts.tables, self._starts
        else:
            prefixes, prefix_tables, starts = prefix, self.prompts.tables.index_select(0, slots), self._single[: n + 1]
        plan = self._plan(lengths, 1, tables, prefix_lengths=prefixes, max_prefix_pages=prefix_tables.shape[1], group_starts=starts)
        return CacheStep(self, torch.where(inside, positions.int(), -1), at, plan, tables, prefix_tables)

    def _plan(self, lengths, queries, tables, **groups) -> AttentionPlan:
        return self.backend.plan(lengths, queries=queries, heads=self.heads, kv_heads=self.kv_heads, head_dim=self.head_dim,
                                 page_size=self.page_size, max_pages=tables.shape[1], **groups)

    def beam_states(self) -> list[BeamState]:
        """The continuations, as ``prepare_reorder`` takes them, for this cache's number of beams: ``max_tokens`` long,
        with lengths of tokens behind the prompt."""
        slots = self.requests * self.beams
        return [BeamState(t[:, self.prompt_pages :].unflatten(1, (slots, -1)).flatten(2, 3)[:, :, : self.max_tokens], slot_dim=1,
                          length_dim=2, beams=self.beams) for t in (self.keys, self.values)]


__all__ = ["CacheStep", "SharedPromptCache"]
