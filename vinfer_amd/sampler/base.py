"""The sampler op family: its interface and its registry.

``sample`` keeps the engine's per-token call unchanged (src/vinfer/runtime/sampler.py:68,
called from runtime/generate.py:129): one 1-D ``[V]`` logits row in the model dtype, the
request's ``SamplingParams``, its seed and the token position, returning a Python ``int``.
Batched entry points are new methods of the interface, as the engine's convention for kernel
families prescribes (kernels/gdn/base.py:7-8). Logits are caller-owned and never written.
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import Protocol

import torch

from vinfer_amd.registry import BackendRegistry
from vinfer_amd.sampler.beams import BeamState
from vinfer_amd.sampling import PackedParams, SamplingParams, penalized


class SamplerBackend(Protocol):
    def sample(
        self,
        logits: torch.Tensor,
        params: SamplingParams,
        seed: int,
        position: int,
        history: Sequence[int] | torch.Tensor | None = None,
    ) -> int:
        """One token id from ``logits`` (``[V]``) for the token at ``position``. ``history`` is
        the request's token ids so far (empty for the first token): it is required when a
        penalty is on (``ValueError`` if it is ``None``), since the penalties are computed from
        it, and ignored otherwise."""
        ...

    def sample_batch(
        self,
        logits: torch.Tensor,
        params: PackedParams,
        uniforms: torch.Tensor,
        hist_ids: torch.Tensor | None = None,
        hist_offsets: torch.Tensor | None = None,
        draft_ids: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor | None]:
        """One token per row of ``logits`` ``[B, V]``: ids int32 ``[B]`` and, when ``draft_ids``
        (int32 ``[B]``) is given, the final probability of each draft id (fp32 ``[B]``).
        ``uniforms`` fp32 ``[B]`` in [0, 1). Histories (int32) are in CSR form (``hist_offsets``
        ``[B + 1]``) or per-row ranges (``hist_offsets`` ``[B, 2]``: row b's ids are
        ``hist_ids[start_b:end_b]``; ranges of different rows must not overlap)."""
        ...

    def probs(
        self,
        logits: torch.Tensor,
        params: PackedParams,
        hist_ids: torch.Tensor | None = None,
        hist_offsets: torch.Tensor | None = None,
    ) -> torch.Tensor:
        """The fp32 ``[B, V]`` distribution ``sample_batch`` draws from (``filtered_probs``,
        sampler.py:50-65, plus penalties and min-p)."""
        ...

    def verify(
        self,
        target_logits: torch.Tensor,
        draft_logits: torch.Tensor,
        draft_tokens: torch.Tensor,
        params: PackedParams,
        u_accept: torch.Tensor,
        u_residual: torch.Tensor,
        u_bonus: torch.Tensor,
        draft_params: PackedParams | None = None,
        draft_states: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """Speculative-decoding verify of ``K`` drafted tokens per sequence: draft ``j`` is
        accepted when ``u_accept[b, j] * q < p`` (``p``, ``q``: the target's and the draft's
        final probabilities of it); at the first rejection the token is drawn with
        ``u_residual[b, j]`` from ``max(0, p - q)`` over ascending ids; with every draft
        accepted, the target's draw at position ``K`` (uniform ``u_bonus[b]``) is added.
        ``target_logits`` ``[B, K + 1, V]``, ``draft_logits`` ``[B, K, V]`` (same dtype),
        ``draft_tokens`` int32 ``[B, K]``, uniforms fp32; ``params`` (one row per sequence)
        apply to the target rows, ``draft_params`` (default: the same) to the draft rows;
        penalties are not applied. A backend with ``sample_states`` (an optional method: the
        draws plus each row's opaque sampling state) takes the drafts' saved states as
        ``draft_states`` ``[B, K, ...]`` instead of sampling the draft rows again. Returns
        ``tokens`` int32 ``[B, K + 1]`` (emitted tokens, then -1) and ``counts`` int32 ``[B]``
        (1 .. K + 1)."""
        ...

    def logprobs(
        self, logits: torch.Tensor, tokens: torch.Tensor | None = None, n_top: int = 0
    ) -> tuple[torch.Tensor | None, torch.Tensor, torch.Tensor]:
        """Log-probabilities of the raw logits ``[B, V]`` (log-softmax before penalties,
        temperature and filters: what ``logprobs`` / ``top_logprobs`` report): of ``tokens``
        (int32 ``[B]``, NaN outside the vocabulary) and of each row's ``n_top`` (0 .. 32)
        largest logits, descending with ties by ascending id. Returns ``(token_logprobs fp32
        [B] or None, top_ids int32 [B, n_top], top_logprobs fp32 [B, n_top])``; a row whose max
        logit is not finite reports NaN."""
        ...

    def penalized_logits(
        self,
        logits: torch.Tensor,
        params: PackedParams,
        hist_ids: torch.Tensor | None = None,
        hist_offsets: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """Penalised fp32 logits ``[B, V]`` and the history count of every id (int32 ``[B, V]``)."""
        ...

    def beam_select(
        self,
        logits: torch.Tensor,
        scores: torch.Tensor,
        n: int,
        finished: torch.Tensor | None = None,
        pad_id: int = 0,
        keep_slots: bool = False,
    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """One step of a beam search: each request's ``n`` (1 .. 64) best continuations over its beams and
        the whole vocabulary, by ``scores[b, w] + log_softmax(logits[b, w])[v]``. ``logits`` ``[B, W, V]``
        (bf16 or fp32, unit stride along V; rows may be shared, as by ``expand``), ``scores`` fp32
        ``[B, W]``, W up to 64. Scores are compared in fp64 (on the hip backend the small terms of a row's sum of
        exponentials are fp32: its log is off by at most 46 2^-23). Equal scores go by ascending beam, then descending logit, then ascending
        id. A beam marked in ``finished`` (bool ``[B, W]``) has one continuation: ``pad_id``, at its own
        score. A beam whose score is not finite has none (the first step: all scores but one -inf), nor has
        a row with a NaN, a +inf or no finite logit, nor a logit of -inf. With ``keep_slots`` (n = W) the
        best child of each parent is placed where the parent is, the others in the free places in their
        order, so that few states move. Returns ``(scores fp32, beams int32, tokens int32)``, ``[B, n]``
        each; where there are fewer continuations, -inf, -1 and -1."""
        ...

    def prepare_reorder(self, states: Sequence[BeamState], requests: int, beams: int):
        """A reusable reordering, in place, of the ``requests * beams`` slots (beams up to 32) of every
        state: ``launch(parents int32 [requests, beams], lengths int32 [requests] or None)`` on the result
        gives slot ``b * beams + w`` what slot ``b * beams + parents[b, w]`` held, up to ``lengths[b]``
        positions (clamped to the state's) in states with a ``length_dim``; a parent outside
        ``[0, beams)`` (the -1 of ``beam_select``) leaves its slot as it is. A HIP graph that captured a launch holds
        addresses: the plan and the states have to outlive it."""
        ...


def require_history(params: SamplingParams, history) -> None:
    """``ValueError`` when ``params`` turns a penalty on and no history was passed: the engine's
    per-token call (src/vinfer/runtime/generate.py:129) passes none, and silently sampling
    without the penalties would be a fallback (kernels/registry.py:5-7 rules those out)."""
    if penalized(params) and history is None:
        raise ValueError(
            "repetition/presence/frequency penalties need the request's token history: "
            "pass history= (the token ids so far, empty for the first token)"
        )


SAMPLER: BackendRegistry[SamplerBackend] = BackendRegistry("sampler")
