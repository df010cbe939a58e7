"""The distillation op family: its interface and its registry.

For each row t, with z = student / temperature, q = softmax(z) and the teacher's entries ``ids[t]``:

- without ``tail``, ``teacher`` holds logits and p = softmax(teacher / temperature) over the row's entries;
- with ``tail``, ``teacher`` holds log-probabilities, p = exp(teacher), and rest = max(0, 1 - sum p) is the
  teacher's share of the ids that are not listed, which the student is held to as a whole.

    loss[t] = weights[t] (sum_k p_k (log p_k - log q_k) + rest (log rest - log q_rest))
    grad[t] = d loss[t] / d student[t], in the student's dtype

``student`` is ``[T, V]`` (bf16 or fp32, unit stride along V), ``ids`` int32 ``[T, K]`` (K up to 1024,
distinct in a row; an id outside ``[0, V)``, as -1, is no entry), ``teacher`` fp32 ``[T, K]``, ``weights``
fp32 ``[T]`` or None (1), the temperature between 1e-6 and 1e6. The hip backend refuses a call of more than 2^24 - 1 segments
(16384 bf16 or 8192 fp32 logits of a row each, fewer in small calls). A row of weight 0 is not read: its loss and gradient are 0. So
are those of a row without entries, whatever its logits hold. An entry of probability 0 adds nothing to the loss; an id of q 0 with p > 0 makes it
infinite. So does, with ``tail``, a rest above 0 (a rounding of the teacher's log-probabilities is enough) where the student allows no
unlisted id: such lists are complete, and ``tail=False`` is theirs.

A row's numbers are sums of fp32 exponentials in an order of their own route: ``loss``, ``loss_and_grad`` and
``loss_and_states`` may differ in their last bits, each of them gives the same bits every time.
"""

from __future__ import annotations

from typing import Protocol

import torch

from vinfer_amd import _vops
from vinfer_amd.registry import BackendRegistry

DTYPES = {torch.bfloat16: _vops.VOPS_BF16, torch.float32: _vops.VOPS_F32}


class DistillBackend(Protocol):
    def loss(self, student: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, weights: torch.Tensor | None = None,
             *, temperature: float = 1.0, tail: bool = False) -> torch.Tensor:
        """The rows' losses, fp32 ``[T]``."""
        ...

    def loss_and_grad(self, student: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor,
                      weights: torch.Tensor | None = None, *, temperature: float = 1.0,
                      tail: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows' losses and the gradient of their sum, ``[T, V]``."""
        ...

    def loss_and_states(self, student: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor,
                        weights: torch.Tensor | None = None, *, temperature: float = 1.0,
                        tail: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows' losses, and what ``grad`` needs beside the student (opaque, ``2 + K`` numbers a row)."""
        ...

    def grad(self, student: torch.Tensor, ids: torch.Tensor, states: torch.Tensor, weights: torch.Tensor | None = None,
             *, temperature: float = 1.0) -> torch.Tensor:
        """The gradient of the losses' sum under ``weights`` (a backward pass: the loss's weights times the
        incoming gradients), from the states of the same student, ids and temperature."""
        ...


def check(student, ids, teacher, weights, temperature) -> None:
    """``ValueError`` for arguments that do not fit together."""
    if student.dtype not in DTYPES:
        raise ValueError(f"distillation supports bf16 and fp32 logits, got {student.dtype}")
    if student.dim() != 2 or (student.stride(1) != 1 and student.shape[1] != 1):
        raise ValueError("student must be [T, V] with unit stride along V")
    T, V = student.shape
    dev = student.device
    if not 1 <= V <= _vops.MAX_VOCAB:
        raise ValueError(f"vocab must be in [1, {_vops.MAX_VOCAB}], got {V}")
    if ids.dtype != torch.int32 or ids.dim() != 2 or ids.shape[0] != T or ids.device != dev:
        raise ValueError(f"ids must be an int32 [{T}, K] tensor on {dev}")
    K = ids.shape[1]
    if not 1 <= K <= _vops.MAX_ENTRIES:
        raise ValueError(f"a row must have 1 to {_vops.MAX_ENTRIES} entries, got {K}")
    if teacher is not None and (teacher.dtype != torch.float32 or teacher.shape != (T, K) or teacher.device != dev):
        raise ValueError(f"teacher must be a float32 [{T}, {K}] tensor on {dev}")
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != (T,) or weights.device != dev):
        raise ValueError(f"weights must be a float32 [{T}] tensor on {dev}")
    low, high = _vops.TEMPERATURES
    if not low <= temperature <= high:
        raise ValueError(f"temperature must be in [{low}, {high}], got {temperature}")


def check_states(states, ids, student) -> None:
    shape = (ids.shape[0], 2 + ids.shape[1])
    if states.dtype != torch.float32 or states.shape != shape or states.device != student.device or not states.is_contiguous():
        raise ValueError(f"states must be the contiguous float32 {list(shape)} tensor of loss_and_states on {student.device}")


DISTILL: BackendRegistry[DistillBackend] = BackendRegistry("distill")
