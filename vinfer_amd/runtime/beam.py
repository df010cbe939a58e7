"""Beam search over a decode model: all requests' beams go through one model step, one selection and one reordering
of their states an iteration. The engine decodes by sampling alone (src/vinfer/runtime/generate.py:105-146).

Request b's beam w has slot ``b * width + w`` of the model. A prompt is prefilled once, into the request's first
slot; the others take its state. From then on a step keeps, of each request's continuations, the ``width`` best
(``beam_select`` with ``keep_slots``: a beam's best child stays where it is), and the states of the slots that change
beams follow (``prepare_reorder``, in place). A beam that draws an end token is finished: it competes at its score
and its slot's steps are not used. Scores are sums of log-probabilities; the results are ordered by
score / length ** length_penalty.

The histories of the tokens are a state like the model's. Nothing waits for the GPU but the test whether every beam
is finished, every ``check_every`` steps.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from dataclasses import dataclass
from typing import Protocol

import torch

from vinfer_amd.sampler.base import SamplerBackend
from vinfer_amd.sampler.beams import BeamState


class BeamModel(Protocol):
    """A decode model whose slots' states can be moved: ``DecodeModel``'s two calls, and the states."""

    device: torch.device

    def prefill(self, slot: int, prompt_ids: torch.Tensor) -> torch.Tensor:
        """Logits ``[V]`` behind the prompt, whose state goes to ``slot``."""
        ...

    def decode(self, slots: torch.Tensor, tokens: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Logits ``[n, V]`` behind one token a slot, whose states move on."""
        ...

    def beam_states(self, slots: int) -> Sequence[BeamState]:
        """The states of slots 0 .. slots - 1 (none: a model without state)."""
        ...


@dataclass(frozen=True)
class Hypothesis:
    tokens: list[int]  # without the prompt; an end token, if one ended it, is the last
    score: float  # the sum of the log-probabilities
    finished: bool


def beam_search(model: BeamModel, sampler: SamplerBackend, prompts: Sequence[Sequence[int]], *, width: int,
                max_tokens: int, eos_token_ids: Sequence[int] = (), length_penalty: float = 1.0,
                check_every: int = 8) -> list[list[Hypothesis]]:
    """Each prompt's ``width`` best continuations of up to ``max_tokens`` tokens, the best first."""
    if not prompts or not all(len(p) for p in prompts):
        raise ValueError("beam_search needs at least one prompt, and no empty one")
    if max_tokens < 1 or check_every < 1:
        raise ValueError(f"max_tokens and check_every must be positive, got {max_tokens} and {check_every}")
    B, W, dev = len(prompts), width, model.device
    lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
    history = torch.zeros(B * W, max_tokens, dtype=torch.int32, device=dev)
    model_states = list(model.beam_states(B * W))
    states = sampler.prepare_reorder(model_states, B, W) if model_states else None
    histories = sampler.prepare_reorder([BeamState(history)], B, W)
    eos = torch.tensor(sorted(set(eos_token_ids)), dtype=torch.int32, device=dev)
    slots = torch.arange(B * W, device=dev)
    own = torch.arange(W, dtype=torch.int32, device=dev).expand(B, W)

    rows = torch.stack([model.prefill(b * W, torch.as_tensor(p, device=dev)) for b, p in enumerate(prompts)])
    logits = rows[:, None].expand(B, W, rows.shape[-1])
    if states is not None:  # (every beam starts from its request's prompt)
        states.launch(torch.zeros(B, W, dtype=torch.int32, device=dev), lengths)
    scores = torch.full((B, W), -math.inf, device=dev)
    scores[:, 0] = 0.0
    finished = torch.zeros(B, W, dtype=torch.bool, device=dev)
    count = torch.zeros(B, W, dtype=torch.int32, device=dev)  # tokens of each beam

    for step in range(max_tokens):
        scores, beams, tokens = sampler.beam_select(logits, scores, W, finished=finished, pad_id=0, keep_slots=True)
        parents = torch.where(beams < 0, own, beams).long()
        histories.launch(beams)
        finished = torch.gather(finished, 1, parents)
        count = torch.gather(count, 1, parents) + (~finished).int()
        history[:, step] = torch.where(finished, 0, tokens).reshape(-1)
        finished = finished | torch.isin(tokens, eos) | (beams < 0)
        if step + 1 == max_tokens or (step + 1) % check_every == 0 and bool(finished.all()):
            break
        if states is not None:
            states.launch(beams, lengths + step)
        positions = (lengths + step).repeat_interleave(W)
        logits = model.decode(slots, tokens.clamp(min=0).reshape(-1).long(), positions.long()).view(B, W, -1)

    out = []
    for b in range(B):
        found = []
        for w in range(W):
            if not math.isfinite(float(scores[b, w])):
                continue
            ids = history[b * W + w, : int(count[b, w])].tolist()
            found.append(Hypothesis(ids, float(scores[b, w]), bool(finished[b, w])))
        found.sort(key=lambda h: -h.score / max(1, len(h.tokens)) ** length_penalty)
        out.append(found)
    return out


__all__ = ["BeamModel", "Hypothesis", "beam_search"]
