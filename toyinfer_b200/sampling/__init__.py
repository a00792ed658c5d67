"""Sampling options and the sampler."""
from .params import GREEDY, BeamParams, SamplingParams
from .sampler import Sampler

__all__ = ["GREEDY", "BeamParams", "SamplingParams", "Sampler"]
