from .sampler import Sampler, SamplingParams, next_rand, stream_seed  # noqa: F401
from .scores import TokenScores, log_probs  # noqa: F401
