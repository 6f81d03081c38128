"""The end of a serving loop: one token per row of logits (csrc/sampling.hip)."""
from __future__ import annotations

from .ssm import _call


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """logits (B,V), V up to 2^20, u (B) random numbers in [0, 1) -> (tokens (B) int64, logprobs (B) fp32).

    temperature, top_k, top_p and min_p are numbers or tensors (B) with a setting per row.  The likeliest token has weight 1, the
    others exp((logit - max) / temperature), rounded to whole 2^-31ths (one below 2^-32 is never drawn); tokens stand in the order of that exponent, ties by
    index.  Kept are the first top_k tokens (0 or less: all), of those the ones of weight min_p or more, of those the shortest
    beginning with a share top_p of their weight (always the first); the token drawn is the first, by index, at which the sum of the
    kept weights passes u times their total.  logprobs: the logs of the probabilities they were drawn with.

    A tensor top_k is read in 32 bits.  A temperature below 1e-6 takes the likeliest token.  NaN counts as -infinity; a row of nothing else gives token -1 and
    -infinity.  The sums are of whole numbers, so a token depends on its row, u and settings alone.  Without autograd only (logits that want a
    gradient are refused: the logprobs would have none)."""
    return _call("sample", logits, u, temperature, top_k, top_p, min_p)
