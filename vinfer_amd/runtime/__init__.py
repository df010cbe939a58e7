"""Callers of the operators: the continuous-batching decode loop, beam search, and the paged cache of their models."""

from vinfer_amd.runtime.batch import BatchDecoder, DecodeModel, NoRoom, SpeculativeDecoder, Step, TextStream, check_request
from vinfer_amd.runtime.beam import BeamModel, Hypothesis, beam_search
from vinfer_amd.runtime.paged import CacheStep, SharedPromptCache

__all__ = ["BatchDecoder", "BeamModel", "CacheStep", "DecodeModel", "Hypothesis", "NoRoom", "SharedPromptCache", "SpeculativeDecoder",
           "Step", "TextStream", "beam_search", "check_request"]
