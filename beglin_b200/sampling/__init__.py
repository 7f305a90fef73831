from .rules import LogitRules
from .sampler import Sampler, SamplingParams, request_key, uniform

__all__ = ["LogitRules", "Sampler", "SamplingParams", "request_key", "uniform"]
