"""``distill_loss``: the distillation loss as a function that torch differentiates in the student's logits."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from vinfer_amd.distill.base import DISTILL, DistillBackend
from vinfer_amd.registry import BackendContext


class _DistillLoss(torch.autograd.Function):
    # The forward pass keeps the student and 2 + K numbers a row; the backward pass reads the student once more
    # and writes the gradient, so nothing of the vocabulary's size lives in between.
    @staticmethod
    def forward(ctx, student, ids, teacher, weights, temperature, tail, backend):
        loss, states = backend.loss_and_states(student, ids, teacher, weights, temperature=temperature, tail=tail)
        ctx.save_for_backward(student, ids, states, weights)
        ctx.temperature, ctx.backend = temperature, backend
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        student, ids, states, weights = ctx.saved_tensors
        # (a row of weight 0 has states of 0, and gradient 0 also where what comes in is infinite or NaN)
        w = g.float() if weights is None else weights * g
        return ctx.backend.grad(student, ids, states, w.contiguous(), temperature=ctx.temperature), *([None] * 6)


def distill_loss(
    student: torch.Tensor,
    ids: torch.Tensor,
    teacher: torch.Tensor,
    weights: torch.Tensor | None = None,
    *,
    temperature: float = 1.0,
    tail: bool = False,
    backend: str | DistillBackend = "hip",
) -> torch.Tensor:
    """The rows' losses (fp32 ``[T]``; see ``DistillBackend``), differentiable in ``student``. ``teacher``
    and ``weights`` are constants. Backward mode alone: an argument with a tangent (forward mode) is refused. ``backend``:
    a name of the ``distill`` family, or a resolved backend."""
    if teacher.requires_grad or (weights is not None and weights.requires_grad):
        raise ValueError("distill_loss differentiates in the student's logits only")
    # (a level is entered: 1.3 us a tensor otherwise)
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (student, teacher, weights)):
        raise ValueError("distill_loss has no forward-mode derivative")
    if isinstance(backend, str):
        backend = DISTILL.resolve(backend, BackendContext(student.device, student.dtype))
    if not (student.requires_grad and torch.is_grad_enabled()):
        return backend.loss(student, ids, teacher, weights, temperature=temperature, tail=tail)
    return _DistillLoss.apply(student, ids, teacher, weights, temperature, tail, backend)


__all__ = ["distill_loss"]
