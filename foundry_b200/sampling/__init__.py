"""Sampling: parameters, the device selector, and its host restatement."""
from .params import SamplingParams, is_ruled, params_of_rows
from .sampler import Sampler, gumbel_scores, stream_key, uniform24

__all__ = ["SamplingParams", "is_ruled", "params_of_rows", "Sampler", "gumbel_scores", "stream_key", "uniform24"]
