"""Beam search's operators: which continuations a step keeps (``beam_select``) and the states of the
search's slots in their parents' order (``prepare_reorder``). The engine decodes one sequence at a time
(src/vinfer/runtime/generate.py:105-146) and has no counterpart.

The checks and layouts here serve both backends; ``select_reference`` and ``ReorderReference`` are the torch
forms, ``HipBeams`` and ``HipReorder`` the ones on the kernels of ``libvops.so``.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence
from dataclasses import dataclass

import torch

from vinfer_amd import _vops

_DTYPES = {torch.bfloat16: _vops.VOPS_BF16, torch.float32: _vops.VOPS_F32}


@dataclass(frozen=True)
class BeamState:
    """One tensor of states that a search's beams carry: ``slot_dim`` indexes the ``requests * beams`` slots
    (request b's beam w in slot ``b * beams + w``); with ``length_dim`` (a cache's or a history's positions)
    only a request's first positions count. Any dtype, any strides without overlap, and no memory that another state
    of the same plan holds."""

    tensor: torch.Tensor
    slot_dim: int = 0
    length_dim: int | None = None


# ---- checks ---------------------------------------------------------------------------------------------
def check_select(logits, scores, n, finished, pad_id, keep_slots) -> None:
    """``ValueError`` for arguments of ``beam_select`` that do not fit together."""
    if logits.dim() != 3 or (logits.stride(2) != 1 and logits.shape[2] != 1):
        raise ValueError("logits must be [B, W, V] with unit stride along V")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"beam_select supports bf16 and fp32 logits, got {logits.dtype}")
    B, W, V = logits.shape
    if B > 65535:
        raise ValueError(f"at most 65535 requests, got {B}")
    if not 1 <= W <= _vops.MAX_BEAMS:
        raise ValueError(f"beams must be in [1, {_vops.MAX_BEAMS}], got {W}")
    if not 1 <= V <= _vops.MAX_VOCAB:
        raise ValueError(f"vocab must be in [1, {_vops.MAX_VOCAB}], got {V}")
    if not 1 <= n <= _vops.MAX_CONTINUATIONS:
        raise ValueError(f"n must be in [1, {_vops.MAX_CONTINUATIONS}], got {n}")
    if keep_slots and n != W:
        raise ValueError(f"keep_slots needs as many continuations as beams, got n {n} and {W} beams")
    if not -(1 << 31) <= pad_id < 1 << 31:
        raise ValueError(f"pad_id must be an int32, got {pad_id}")
    if scores.dtype != torch.float32 or scores.shape != (B, W) or scores.device != logits.device:
        raise ValueError(f"scores must be a float32 [{B}, {W}] tensor on {logits.device}")
    if finished is not None and (finished.dtype != torch.bool or finished.shape != (B, W)
                                 or finished.device != logits.device):
        raise ValueError(f"finished must be a bool [{B}, {W}] tensor on {logits.device}")


def _apart(a: int, da: Sequence[tuple[int, int]], b: int, db: Sequence[tuple[int, int]]) -> bool:
    """Whether the bytes at ``a + sum(i * stride)`` over the (stride, extent) pairs ``da`` are shown to be none of
    ``b``'s: their ranges do not meet, or they do not within one period of a stride that the outer dimensions of both
    are multiples of."""
    end_a, end_b = (x + sum(st * (n - 1) for st, n in d) + 1 for x, d in ((a, da), (b, db)))
    if end_a <= b or end_b <= a:
        return True
    for period in sorted({st for d in (da, db) for st, _ in d if st > 1}, reverse=True):
        inner = [[(st, n) for st, n in d if st % period] for d in (da, db)]
        if len(inner[0]) + len(inner[1]) == len(da) + len(db):
            continue
        for origin in {a, b}:
            at = [(x - origin) % period for x in (a, b)]
            if all(x + sum(st * (n - 1) for st, n in d) < period for x, d in zip(at, inner)) \
                    and _apart(at[0], inner[0], at[1], inner[1]):
                return True
    return False


def check_states(states: Sequence[BeamState], requests: int, beams: int) -> torch.device:
    """``ValueError`` for states that ``prepare_reorder`` cannot take; the states' device."""
    if not states:
        raise ValueError("prepare_reorder needs at least one state")
    if requests < 0 or not 1 <= beams <= _vops.MAX_REORDER_BEAMS:
        raise ValueError(f"requests must be >= 0 and beams in [1, {_vops.MAX_REORDER_BEAMS}], got {requests} and {beams}")
    dev = states[0].tensor.device
    spans, layouts = [], {}
    for i, s in enumerate(states):
        t = s.tensor
        if t.device != dev:
            raise ValueError(f"states must be on one device, got {dev} and {t.device}")
        if t.requires_grad:
            raise ValueError(f"state {i} requires a gradient: states are reordered in place")
        if not 0 <= s.slot_dim < t.dim() or t.shape[s.slot_dim] != requests * beams:
            raise ValueError(f"state {i}: dimension {s.slot_dim} of {tuple(t.shape)} must hold the {requests * beams} slots")
        if s.length_dim is not None and (not 0 <= s.length_dim < t.dim() or s.length_dim == s.slot_dim):
            raise ValueError(f"state {i}: length_dim {s.length_dim} is not another dimension of {tuple(t.shape)}")
        if t.numel() == 0:
            continue
        dims = sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1)
        end = 1
        for st, n in dims:
            if st < end:
                raise ValueError(f"state {i}: elements of a tensor with strides {t.stride()} may overlap")
            end = st * (n - 1) + end
        size = t.element_size()
        d = tuple((st * size, n) for st, n in dims) + ((1, size),)
        spans.append((t.data_ptr(), i, layouts.setdefault(d, len(layouts)), t.data_ptr() + end * size))
    # One launch moves all states, in no order: what two of them held would be read and written at once. (Views of one
    # buffer differ by few offsets: each is looked at once.)
    spans.sort()
    layout, known = list(layouts), {}
    for k, (p, i, d, end) in enumerate(spans):
        for q, j, e, _ in spans[k + 1 :]:
            if q >= end:
                break
            apart = known.get((q - p, d, e))
            if apart is None:
                apart = known[q - p, d, e] = _apart(0, layout[d], q - p, layout[e])
            if not apart:
                raise ValueError(f"states {min(i, j)} and {max(i, j)} may hold the same memory")
    return dev


def check_reorder(parents, lengths, requests, beams, dev, has_length) -> None:
    if parents.dtype != torch.int32 or parents.shape != (requests, beams) or parents.device != dev:
        raise ValueError(f"parents must be an int32 [{requests}, {beams}] tensor on {dev}")
    if lengths is None:
        if has_length:
            raise ValueError("lengths must be given: a state has a length_dim")
    elif lengths.dtype != torch.int32 or lengths.shape != (requests,) or lengths.device != dev:
        raise ValueError(f"lengths must be an int32 [{requests}] tensor on {dev}")


def describe(s: BeamState) -> _vops.VopsState:
    """The library's description of a state: what is contiguous in a slot makes runs, the rest are outer
    dimensions (at most three). Positions join the run behind them where it is whole."""
    t, size = s.tensor, s.tensor.element_size()
    # (stride and extent of each dimension but the slots', the innermost first)
    dims = sorted((st * size, -i, n, i == s.length_dim) for i, (st, n) in enumerate(zip(t.stride(), t.shape))
                  if i != s.slot_dim and (n > 1 or i == s.length_dim))
    run, unit, length_at = size, 0, -1
    outer: list[list] = []  # [stride, extent, is the length]
    for st, _, n, is_length in dims:
        if not outer and length_at < 0 and (st == run or n == 1):
            if is_length:
                unit, length_at = run, 3
            run *= n
        elif outer and not is_length and not outer[-1][2] and st == outer[-1][0] * outer[-1][1]:
            outer[-1][1] *= n
        else:
            outer.append([st, n, is_length])
    if max([t.shape[s.length_dim] if s.length_dim is not None else 0] + [n for _, n, _ in outer]) >= 1 << 31:
        raise ValueError(f"a state of shape {tuple(t.shape)} has a dimension past 2^31")
    if len(outer) > 3:
        raise ValueError(f"a state of shape {tuple(t.shape)} and strides {t.stride()} has more than three strided dimensions")
    d = _vops.VopsState()
    d.data = t.data_ptr()
    d.slot_stride = t.stride(s.slot_dim) * size
    d.run, d.unit = run, unit
    d.length_dim = length_at
    d.max_length = t.shape[s.length_dim] if s.length_dim is not None else 0
    for i in range(3):  # (the outermost first)
        d.size[i], d.stride[i] = 1, 0
    for i, (st, n, is_length) in enumerate(reversed(outer)):
        at = 3 - len(outer) + i
        d.size[at], d.stride[at] = n, st
        if is_length:
            d.length_dim = at
    return d


# ---- torch ----------------------------------------------------------------------------------------------
def select_reference(logits, scores, n, finished=None, pad_id=0, keep_slots=False):
    """``SamplerBackend.beam_select`` in torch, a request at a time."""
    check_select(logits, scores, n, finished, pad_id, keep_slots)
    B, W, V = logits.shape
    out_scores = torch.full((B, n), -math.inf)
    out_beams = torch.full((B, n), -1, dtype=torch.int32)
    out_tokens = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):
        entries = []  # (score, -beam, logit, -id, token)
        for w in range(W):
            score = float(scores[b, w])
            if not math.isfinite(score):
                continue
            if finished is not None and bool(finished[b, w]):
                entries.append((score, -w, 0.0, 0, pad_id))
                continue
            x = logits[b, w].double().cpu()
            m = x.max()  # (NaN where there is one)
            if not bool(torch.isfinite(m)):
                continue
            logs = torch.log(torch.exp(x - m).sum())
            order = torch.sort(x + 0.0, descending=True, stable=True).indices[:n]
            entries += [(float(c), -w, float(x[v]) + 0.0, -int(v), int(v))
                        for v, c in zip(order, (x[order] - m) - logs + score) if float(c) > -math.inf]
        entries.sort(reverse=True)
        chosen = entries[:n]
        places = list(range(n))
        if keep_slots:
            first: dict[int, int] = {}
            for i, e in enumerate(chosen):
                first.setdefault(-e[1], i)
            free = iter([k for k in range(n) if k not in first])
            stays = {i: w for w, i in first.items()}
            places = [stays[i] if i in stays else next(free) for i in range(n)]
        for i, e in enumerate(chosen):
            out_scores[b, places[i]], out_beams[b, places[i]], out_tokens[b, places[i]] = e[0], -e[1], e[4]
    dev = logits.device
    return out_scores.to(dev), out_beams.to(dev), out_tokens.to(dev)


class ReorderReference:
    """``SamplerBackend.prepare_reorder`` in torch."""

    def __init__(self, states: Sequence[BeamState], requests: int, beams: int) -> None:
        self.states, self.requests, self.beams = list(states), requests, beams
        self.device = check_states(states, requests, beams)
        self._has_length = any(s.length_dim is not None for s in states)

    def launch(self, parents: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        check_reorder(parents, lengths, self.requests, self.beams, self.device, self._has_length)
        own = torch.arange(self.beams, device=self.device)
        p = torch.where((parents >= 0) & (parents < self.beams), parents, own)
        source = (torch.arange(self.requests, device=self.device)[:, None] * self.beams + p).reshape(-1)
        for s in self.states:
            t = s.tensor
            new = t.index_select(s.slot_dim, source)
            if s.length_dim is not None:
                shape = [1] * t.dim()
                shape[s.slot_dim], shape[s.length_dim] = t.shape[s.slot_dim], t.shape[s.length_dim]
                inside = torch.arange(t.shape[s.length_dim], device=self.device) < lengths.repeat_interleave(self.beams)[:, None]
                if s.length_dim < s.slot_dim:
                    inside = inside.T
                new = torch.where(inside.reshape(shape), new, t)
            t.copy_(new)


# ---- the kernels ----------------------------------------------------------------------------------------
class HipBeams:
    """The ``hip`` sampler backend's beam selection, on torch's current stream of the logits' device. Outputs and
    workspace are torch's: a call's workspace is reused only behind its work."""

    def __init__(self) -> None:
        self._lib = _vops.load()
        self._need: dict[tuple, int] = {}  # workspace bytes by sizes

    def select(self, logits, scores, n, finished=None, pad_id=0, keep_slots=False):
        check_select(logits, scores, n, finished, pad_id, keep_slots)
        dev = logits.device
        if dev.type != "cuda":
            raise ValueError(f"hip sampler needs logits on a GPU, got {dev}")
        B, W, V = logits.shape
        scores = scores.contiguous()
        out_scores = torch.empty(B, n, dtype=torch.float32, device=dev)
        out_beams = torch.empty(B, n, dtype=torch.int32, device=dev)
        out_tokens = torch.empty(B, n, dtype=torch.int32, device=dev)
        a = _vops.VopsBeamArgs()
        a.logits, a.dtype = logits.data_ptr(), _DTYPES[logits.dtype]
        a.requests, a.beams, a.vocab = B, W, V
        a.request_stride, a.beam_stride = logits.stride(0), logits.stride(1)
        a.scores = scores.data_ptr()
        if finished is not None:
            finished = finished.contiguous()
            a.finished = finished.data_ptr()
        a.n, a.pad_id = n, pad_id
        a.flags = _vops.VOPS_BEAM_KEEP_SLOTS if keep_slots else 0
        a.out_scores, a.out_beams, a.out_tokens = out_scores.data_ptr(), out_beams.data_ptr(), out_tokens.data_ptr()
        sizes = a.dtype, B, W, V, n
        need = self._need.get(sizes)
        if need is None:
            need = self._need[sizes] = self._lib.vops_beam_workspace_bytes(*sizes)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)  # (torch aligns to 512 bytes)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _vops.call(self._lib.vops_beam_select, dev, ctypes.byref(a))
        return out_scores, out_beams, out_tokens


class HipReorder:
    """A reusable reordering of fixed states (``prepare_reorder`` of the ``hip`` sampler backend). It may be dropped as
    soon as its launches are enqueued, on whatever streams; only graphs that captured one need it to live on."""

    def __init__(self, states: Sequence[BeamState], requests: int, beams: int) -> None:
        self._lib = _vops.load()
        self.states, self.requests, self.beams = list(states), requests, beams
        dev = self.device = check_states(states, requests, beams)
        if dev.type != "cuda":
            raise ValueError(f"hip sampler needs states on a GPU, got {dev}")
        if requests > 65535 or len(self.states) > 65535:
            raise ValueError(f"at most 65535 requests and states, got {requests} and {len(self.states)}")
        self._has_length = any(s.length_dim is not None for s in states)
        descs = [describe(s) for s in self.states if s.tensor.numel()]
        self._max = 0
        for d in descs:
            columns = int(self._lib.vops_state_columns(ctypes.byref(d)))
            if columns < 0:
                raise ValueError("a state is too large to be described")
            self._max = max(self._max, columns)
        self._n = len(descs)
        blob = b"".join(bytes(d) for d in descs)
        self._descs = torch.frombuffer(bytearray(blob), dtype=torch.uint8).to(dev) if blob else None
        self._stream = torch._C._cuda_getCurrentRawStream(dev.index)  # (whose memory the descriptions are in)

    def launch(self, parents: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Enqueue one reordering on torch's current stream of the states' device."""
        check_reorder(parents, lengths, self.requests, self.beams, self.device, self._has_length)
        if self._descs is None:
            return
        if torch._C._cuda_getCurrentRawStream(self.device.index) != self._stream:
            self._descs.record_stream(torch.cuda.current_stream(self.device))
        parents = parents.contiguous()
        if lengths is not None:
            lengths = lengths.contiguous()
        _vops.call(self._lib.vops_reorder, self.device, self._descs.data_ptr(), self._n, self._max, self.requests,
                   self.beams, parents.data_ptr(), None if lengths is None else lengths.data_ptr())


__all__ = ["BeamState", "HipBeams", "HipReorder", "ReorderReference", "select_reference"]
