"""Distillation from a teacher's top entries: backends ``reference`` (torch) and ``hip`` (gfx950 kernels), and
``distill_loss``, the loss as a differentiable function."""

from vinfer_amd.distill import hip as _hip  # noqa: F401  (registers "hip")
from vinfer_amd.distill import reference as _reference  # noqa: F401  (registers "reference")
from vinfer_amd.distill.base import DISTILL, DistillBackend
from vinfer_amd.distill.function import distill_loss
from vinfer_amd.distill.hip import HipDistill
from vinfer_amd.distill.reference import ReferenceDistill

__all__ = ["DISTILL", "DistillBackend", "HipDistill", "ReferenceDistill", "distill_loss"]
