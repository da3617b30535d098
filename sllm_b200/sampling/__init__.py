from .params import BeamParams, SamplingParams
from .sampler import Sampler

__all__ = ["BeamParams", "SamplingParams", "Sampler"]
