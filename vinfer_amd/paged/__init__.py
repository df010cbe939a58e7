"""A paged cache that sequences share: page tables on the GPU, rotation and storing, attention of sequences behind
shared prefixes. Backends ``reference`` (torch) and ``hip`` (gfx950 kernels)."""

from vinfer_amd.paged import hip as _hip  # noqa: F401  (registers "hip")
from vinfer_amd.paged import reference as _reference  # noqa: F401  (registers "reference")
from vinfer_amd.paged.base import (
    PAGED,
    AttentionPlan,
    Extension,
    PagedBackend,
    PageTables,
    Rotary,
    rotary_frequencies,
)
from vinfer_amd.paged.hip import HipPaged
from vinfer_amd.paged.reference import ReferencePaged

__all__ = ["PAGED", "AttentionPlan", "Extension", "HipPaged", "PageTables", "PagedBackend", "ReferencePaged", "Rotary",
           "rotary_frequencies"]
