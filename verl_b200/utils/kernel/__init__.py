from .linear_cross_entropy import LinearCrossEntropy, linear_cross_entropy
from .token_logprobs import TokenLogprobs, logprobs_of_logits, token_logprobs

__all__ = ["LinearCrossEntropy", "linear_cross_entropy", "TokenLogprobs", "token_logprobs", "logprobs_of_logits"]
