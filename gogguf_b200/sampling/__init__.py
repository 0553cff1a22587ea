"""Sampling: configuration, host chain, device kernels, and what is done to the logits before."""
from .grammar import TokenGrammar
from .sampler import (FunctionSampler, Sampler, SamplerConfig, apply_repeat_penalty, greedy, make_sampler,
                      sample_host, uniform01)
from .shaping import LogitShaping, shape_host

__all__ = ["FunctionSampler", "Sampler", "SamplerConfig", "make_sampler", "apply_repeat_penalty", "greedy", "sample_host", "uniform01", "TokenGrammar",
           "LogitShaping", "shape_host"]
