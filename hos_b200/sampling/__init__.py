from .sampler import Sampler, SamplingParams, next_rand, stream_seed  # noqa: F401
from .scores import ScoredToken, TokenScores, log_probs, scored_tokens  # noqa: F401
