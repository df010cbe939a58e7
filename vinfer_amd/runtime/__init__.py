"""Callers of the sampler: the continuous-batching decode loop and beam search."""

from vinfer_amd.runtime.batch import BatchDecoder, DecodeModel, SpeculativeDecoder, Step, TextStream, check_request
from vinfer_amd.runtime.beam import BeamModel, Hypothesis, beam_search

__all__ = ["BatchDecoder", "BeamModel", "DecodeModel", "Hypothesis", "SpeculativeDecoder", "Step", "TextStream",
           "beam_search", "check_request"]
