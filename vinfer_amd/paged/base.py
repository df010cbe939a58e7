"""The paged-cache op family: its interface, its registry and the checks that serve both backends.

A cache is two tensors ``[pages, page_size, kv_heads, head_dim]``, keys and values (one pair a layer). Position p of a
sequence lies in page ``table[p // page_size]``, at its place ``p % page_size``; its slot is
``page * page_size + place``. The engine's own cache is contiguous, one sequence a slot
(src/vinfer/state/pool.py:41-128), and has no counterpart of these operators.

A step of a decode model: ``extend`` gives the new tokens their pages, slots and positions, ``plan`` spreads the step's
attention over the chip, and each layer calls ``rotate_store`` and ``attend``; after a verification ``shrink`` takes
back what was refused. Nothing waits for the GPU, so a step can be captured into a graph.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Protocol

import torch
from torch.autograd import forward_ad

from vinfer_amd import _vpaged
from vinfer_amd.registry import BackendRegistry

DTYPES = {torch.bfloat16: _vpaged.VPAGED_BF16, torch.float16: _vpaged.VPAGED_F16}


@dataclass(eq=False, frozen=True)
class PageTables:
    """What each sequence holds, and a stack of the pages that nobody holds, on one device (contiguous int32 tensors):
    ``tables [S, max_pages]``, ``lengths [S]``, ``free [pages]`` whose first ``free_count [1]`` entries are free, the
    last of them taken first. ``extend`` and ``shrink`` change them in place; a caller may too (a sequence that holds
    pages of its own choosing, a table's row that is a view of another's)."""

    tables: torch.Tensor
    lengths: torch.Tensor
    free: torch.Tensor
    free_count: torch.Tensor
    page_size: int

    def __post_init__(self) -> None:
        dev = self.tables.device
        for name, t, dim in (("tables", self.tables, 2), ("lengths", self.lengths, 1), ("free", self.free, 1),
                             ("free_count", self.free_count, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or t.device != dev or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor of {dim} dimension(s) on {dev}")
        S, M = self.tables.shape
        if self.lengths.shape[0] != S or self.free_count.shape[0] != 1:
            raise ValueError(f"lengths must have the tables' {S} sequences and free_count one element")
        if S > _vpaged.MAX_SEQUENCES or M < 1 or self.free.shape[0] < 1 or S * M >= 1 << 31:
            raise ValueError(f"at most {_vpaged.MAX_SEQUENCES} sequences, at least a page, and fewer than 2^31 entries, "
                             f"got {S} sequences, tables of {M} and {self.free.shape[0]} pages")
        check_page_size(self.page_size, self.free.shape[0])

    @classmethod
    def empty(cls, sequences: int, max_pages: int, pages: int, page_size: int, device) -> PageTables:
        """Sequences of no length, and every page free (page 0 is taken first)."""
        mk = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        count = torch.full((1,), pages, dtype=torch.int32, device=device)
        return cls(mk(sequences, max_pages), mk(sequences), free, count, page_size)

    @property
    def device(self) -> torch.device:
        return self.tables.device


@dataclass(eq=False)
class Extension:
    """``extend``'s outputs: of each token (the sequences' one after the other) its slot, its position and its
    sequence, int32, -1 where there is none; and which sequences were served (bool)."""

    slots: torch.Tensor
    positions: torch.Tensor
    sequences: torch.Tensor
    served: torch.Tensor


@dataclass(eq=False, frozen=True)
class Rotary:
    """How queries and keys are turned: pair j of a head's first ``2 * len(frequencies)`` elements by
    ``position * frequencies[j]`` (float64), ``magnitude`` times as long. Pairs are elements (j, j + len) or, where
    ``interleaved``, (2j, 2j + 1)."""

    frequencies: torch.Tensor
    interleaved: bool = False
    magnitude: float = 1.0

    def __post_init__(self) -> None:
        f = self.frequencies
        if f.dtype != torch.float64 or f.dim() != 1 or not f.is_contiguous():
            raise ValueError("frequencies must be a contiguous float64 tensor of one dimension")
        if 2 * f.shape[0] > _vpaged.MAX_HEAD_DIM:
            raise ValueError(f"at most {_vpaged.MAX_HEAD_DIM // 2} frequencies, got {f.shape[0]}")
        if not abs(self.magnitude) <= torch.finfo(torch.float32).max:
            raise ValueError(f"magnitude must be finite in fp32, got {self.magnitude}")


def rotary_frequencies(dim: int, *, base: float = 10000.0, stretch: float = 1.0, trained: int | None = None,
                       turns: tuple[float, float] = (1.0, 32.0), device=None) -> torch.Tensor:
    """``base ** (-2j / dim)`` for j < dim / 2, for contexts ``stretch`` times as long as trained on: without
    ``trained`` every frequency divided by ``stretch``; with it (a number of positions) those that turn at most
    ``turns[0]`` times over it are divided, those that turn at least ``turns[1]`` times stay, and between the two
    they go linearly from one to the other."""
    if dim < 0 or dim % 2 or not base > 0.0 or not stretch > 0.0:
        raise ValueError(f"dim must be even, base and stretch positive, got {dim}, {base}, {stretch}")
    f = base ** -(torch.arange(0, dim, 2, dtype=torch.float64, device=device) / max(dim, 1))
    if trained is None:
        return f / stretch
    low, high = turns
    if trained < 1 or not low < high:
        raise ValueError(f"trained must be positive and turns ascend, got {trained} and {turns}")
    keep = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (1 - keep) * f / stretch + keep * f


@dataclass(eq=False)
class AttentionPlan:
    """``plan``'s result, for the attention of one step: opaque but for the shape that it was made for, which has no type.
    Layers share it; calls on other streams must be ordered behind its making by the caller."""

    sequences: int
    groups: int
    queries: int
    heads: int
    kv_heads: int
    head_dim: int
    page_size: int
    max_pages: int
    max_prefix_pages: int
    device: torch.device
    data: object  # the backend's


class PagedBackend(Protocol):
    """Serving operators: none has a derivative, and arguments that ask for one (a gradient where those are enabled, a
    tangent of forward mode) are refused."""

    def extend(self, pages: PageTables, counts: torch.Tensor, tokens: int) -> Extension:
        """Sequence s grows by ``counts[s]`` positions (int32; below 0: 0), the sequences in their order taking the
        pages they need. A sequence is served whole or not at all: not where its table would be too short, where its
        tokens lie past ``tokens``, or where the pages that it and those before it need are more than are free. One that
        asks for nothing is served, but none behind tokens that lie past ``tokens`` is. The sequences' tokens lie one
        after the other, ``tokens`` places in all."""
        ...

    def shrink(self, pages: PageTables, lengths: torch.Tensor) -> None:
        """Cut sequences to ``lengths`` (int32 ``[S]``; below 0: 0) where they are longer. Their last pages go back,
        in the reverse order of their taking: what one ``extend`` took is laid back as it was."""
        ...

    def rotate_store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                     k_pages: torch.Tensor, v_pages: torch.Tensor, rotary: Rotary) -> torch.Tensor:
        """``q [N, heads, head_dim]`` turned by the tokens' ``positions`` (int32), ``k [N, kv_heads, head_dim]`` turned
        and stored with ``v`` at ``slots`` (int32, distinct; outside the pages: not stored). A token at a position
        below 0 is none: its queries come out 0, and nothing is stored. The rest of the cache keeps its contents."""
        ...

    def plan(self, lengths: torch.Tensor, *, queries: int, heads: int, kv_heads: int, head_dim: int, page_size: int,
             max_pages: int, prefix_lengths: torch.Tensor | None = None, max_prefix_pages: int = 0,
             group_starts: torch.Tensor | None = None) -> AttentionPlan:
        """Spread a step's attention over the chip, from the lengths (int32, on the device): the ``queries`` new tokens
        of each sequence are the last of its ``lengths[s]`` own positions, held in tables of ``max_pages``. With
        ``prefix_lengths [B]`` and ``group_starts [B + 1]`` (ascending from 0 to the sequences' number) sequences
        ``group_starts[g]`` up to ``group_starts[g + 1]`` share a prefix of ``prefix_lengths[g]`` positions, which
        lies before their own. Lengths past the tables are taken as what the tables hold."""
        ...

    def attend(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
               plan: AttentionPlan, *, prefix_tables: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
        """Attention ``[S, queries, heads, head_dim]``: token t of sequence s sees its group's prefix and the own
        positions up to ``lengths[s] - queries + t``; where that is below 0 there is no such token (a batch padded on
        the left, a finished sequence), and its output is 0. Query heads share key heads in order. ``scale`` (in fp32,
        2^-126 to 2^64) defaults to ``head_dim ** -0.5``. What lies behind the lengths is not seen, whatever it holds; a
        value that is not finite at an own position reaches all of the sequence's new tokens of the call. An entry of a
        table outside the cache is taken as the nearest page. Scores are fp32, weights rounded to the values' type. The ``hip`` backend takes ``q`` of any layout with unit stride along its
        heads' elements, and caches of 16-byte aligned rows: strides of multiples of 8 elements, pages less than 2^31
        elements apart, a page's positions (16 at least) within 2^30."""
        ...


# ---- checks ---------------------------------------------------------------------------------------------
def check_page_size(page_size: int, pages: int) -> None:
    if not 1 <= page_size <= _vpaged.MAX_PAGE_SIZE or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two up to {_vpaged.MAX_PAGE_SIZE}, got {page_size}")
    if pages * page_size >= 1 << 31:
        raise ValueError(f"a cache must hold fewer than 2^31 positions, got {pages} pages of {page_size}")


def _words(name: str, t: torch.Tensor, n: int, device) -> None:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device:
        raise ValueError(f"{name} must be an int32 [{n}] tensor on {device}")


def differentiated() -> bool:
    """Whether a forward-mode level is entered, within which tensors may carry tangents (else there is nothing to ask)."""
    return forward_ad._current_level >= 0


def check_constants(what: str, **tensors) -> None:
    """``ValueError`` for an argument that asks for a derivative, in either mode: ``what`` has none."""
    for name, t in tensors.items():
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: {what} has none")
        if differentiated() and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has a tangent: {what} has no forward-mode derivative")


def check_extend(pages: PageTables, counts, tokens: int) -> None:
    _words("counts", counts, pages.lengths.shape[0], pages.tables.device)
    if not 0 <= tokens <= _vpaged.MAX_TOKENS or (tokens and not counts.shape[0]):
        raise ValueError(f"tokens must be in [0, {_vpaged.MAX_TOKENS}], and 0 without sequences, got {tokens}")


def check_shrink(pages: PageTables, lengths) -> None:
    _words("lengths", lengths, pages.lengths.shape[0], pages.tables.device)


def check_cache(k_pages, v_pages, kv_heads: int, head_dim: int, like) -> None:
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dim() != 4 or t.shape[2] != kv_heads or t.shape[3] != head_dim:
            raise ValueError(f"{name} must be [pages, page_size, {kv_heads}, {head_dim}], got {tuple(t.shape)}")
        if t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
        if t.stride(3) != 1 and head_dim > 1:
            raise ValueError(f"{name} must have unit stride along its heads' elements")
    if k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
        raise ValueError("k_pages and v_pages must have one shape and one layout")
    check_page_size(k_pages.shape[1], k_pages.shape[0])


def check_rotate(q, k, v, positions, slots, k_pages, v_pages, rotary: Rotary) -> None:
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q must be [N, heads, D], k and v [N, kv_heads, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    N, _, D = q.shape
    if not 1 <= D <= _vpaged.MAX_HEAD_DIM or max(q.shape[1], k.shape[1]) > _vpaged.MAX_HEADS:
        raise ValueError(f"heads of up to {_vpaged.MAX_HEAD_DIM} elements, at most {_vpaged.MAX_HEADS} of them, "
                         f"got {tuple(q.shape)} and {tuple(k.shape)}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"q, k and v must be of one type on one device, got {t.dtype} on {t.device} for {name}")
        if t.stride(2) != 1 and D > 1 and t.numel():
            raise ValueError(f"{name} must have unit stride along its heads' elements")
    check_constants("rotate_store", q=q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, frequencies=rotary.frequencies)
    _words("positions", positions, N, q.device)
    _words("slots", slots, N, q.device)
    check_cache(k_pages, v_pages, k.shape[1], D, q)
    if rotary.frequencies.device != q.device or 2 * rotary.frequencies.shape[0] > D:
        raise ValueError(f"the rotary must turn at most {D} elements, on {q.device}, got "
                         f"{2 * rotary.frequencies.shape[0]} on {rotary.frequencies.device}")


def check_plan(lengths, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths, max_prefix_pages,
               group_starts) -> None:
    if lengths.dim() != 1 or lengths.shape[0] > _vpaged.MAX_SEQUENCES:
        raise ValueError(f"lengths must have one dimension of up to {_vpaged.MAX_SEQUENCES} sequences")
    _words("lengths", lengths, lengths.shape[0], lengths.device)
    if not 1 <= queries <= _vpaged.MAX_QUERIES:
        raise ValueError(f"queries must be in [1, {_vpaged.MAX_QUERIES}], got {queries}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads or heads > _vpaged.MAX_HEADS:
        raise ValueError(f"heads must be a multiple of kv_heads up to {_vpaged.MAX_HEADS}, got {heads} and {kv_heads}")
    if head_dim % 8 or not 8 <= head_dim <= _vpaged.MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 in [8, {_vpaged.MAX_HEAD_DIM}], got {head_dim}")
    check_page_size(page_size, 0)
    if max_pages < 1:
        raise ValueError(f"max_pages must be positive, got {max_pages}")
    if (prefix_lengths is None) != (group_starts is None):
        raise ValueError("prefix_lengths and group_starts go together")
    if prefix_lengths is not None:
        if prefix_lengths.dim() != 1 or not 1 <= prefix_lengths.shape[0] <= _vpaged.MAX_SEQUENCES:
            raise ValueError(f"prefix_lengths must have one dimension of 1 to {_vpaged.MAX_SEQUENCES} groups")
        _words("prefix_lengths", prefix_lengths, prefix_lengths.shape[0], lengths.device)
        _words("group_starts", group_starts, prefix_lengths.shape[0] + 1, lengths.device)
        if max_prefix_pages < 1:
            raise ValueError(f"max_prefix_pages must be positive with prefixes, got {max_prefix_pages}")


def check_attend(q, k_pages, v_pages, tables, plan: AttentionPlan, prefix_tables, scale) -> None:
    if q.shape != (plan.sequences, plan.queries, plan.heads, plan.head_dim) or q.device != plan.device:
        raise ValueError(f"q must be [{plan.sequences}, {plan.queries}, {plan.heads}, {plan.head_dim}] on {plan.device}, as "
                         f"planned, got {tuple(q.shape)} on {q.device}")
    if q.stride(3) != 1 and q.numel():
        raise ValueError("q must have unit stride along its heads' elements")
    check_constants("attend", q=q, k_pages=k_pages, v_pages=v_pages)
    check_cache(k_pages, v_pages, plan.kv_heads, plan.head_dim, q)
    if k_pages.shape[1] != plan.page_size or (k_pages.shape[0] < 1 and plan.sequences):
        raise ValueError(f"the cache must have pages, of the plan's {plan.page_size} positions, got {tuple(k_pages.shape)}")
    for name, t, n, m in (("tables", tables, plan.sequences, plan.max_pages),
                          ("prefix_tables", prefix_tables, plan.groups, plan.max_prefix_pages)):
        if t is None and name == "prefix_tables" and not plan.groups:
            continue
        if t is None or t.dtype != torch.int32 or t.shape != (n, m) or t.device != q.device or (t.stride(1) != 1 and m > 1):
            raise ValueError(f"{name} must be an int32 [{n}, {m}] tensor with unit stride along its pages on {q.device}")
    if scale is not None and not 2.0**-126 <= scale <= 2.0**64:
        raise ValueError(f"scale must be in [2^-126, 2^64], got {scale}")


PAGED: BackendRegistry[PagedBackend] = BackendRegistry("paged")
