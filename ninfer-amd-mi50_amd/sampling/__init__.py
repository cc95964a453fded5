from .params import SamplingParams
from .sampler import SampleRow, Sampler, TokenLogprob, fresh_seed, uniform

__all__ = ["SamplingParams", "SampleRow", "Sampler", "TokenLogprob", "fresh_seed", "uniform"]
