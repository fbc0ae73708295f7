"""The log-probabilities, entropies and likeliest tokens of given scores in 64
bits on the CPU, and how far a computation in FP32 may be from them."""

import math

import torch


def log_probs(scores, tokens, top=0, temperature=1.0):
    """(logprobs, entropy, ids, best) in 64 bits: the log-softmax of scores /
    temperature at the tokens (0 for a token outside the vocabulary), the
    entropy, the tokens of the `top` largest scores (equal ones the lowest, a NaN
    the largest) with their log-probabilities; NaN where the scores hold a NaN or
    +inf or nothing above -inf."""
    B, T, V = scores.shape
    x = scores.double()
    logs = torch.log_softmax(x / temperature, -1)
    none = torch.isnan(x).any(-1) | ~torch.isfinite(x.amax(-1))
    logs[none] = math.nan
    entropy = -torch.where(logs == -math.inf, 0.0, logs.exp() * logs).sum(-1)
    rank = torch.where(torch.isnan(x), math.inf, x)
    # a NaN above +inf: two stable sorts, the second by what a NaN is
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    nan_first = torch.isnan(x).gather(-1, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    ids = order.gather(-1, nan_first)[..., :top]
    inside = (tokens >= 0) & (tokens < V)
    at = logs.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0]
    return torch.where(inside, at, 0.0), entropy, ids, logs.gather(-1, ids)


def bounds(scores, temperature=1.0):
    """(one, slope, entropy): what FP32 may add to a log-probability, one +
    slope |d| + 2^-24 |logprob| with d = (x - max) / temperature, and to the
    entropy.  In units of 2^-24: d is off by 3 |d| (the difference, the
    reciprocal, the product); an exponential by 5 |d| (d, and the product by
    log2 e) and 4 (exp2 itself, 2 steps of 2^-23); a sum of V terms over at least
    256 threads by V / 256 + 64 of itself; the logarithms by 4 of themselves."""
    x = scores.double()
    V = x.shape[-1]
    d = (x - x.amax(-1, keepdim=True)) / temperature
    p = torch.softmax(x / temperature, -1)
    finite = torch.where(p > 0, d, 0.0).abs()
    mean, square = (p * finite).sum(-1), (p * finite * finite).sum(-1)
    log_sum = torch.logsumexp(d, -1)
    unit = 2.0 ** -24
    adds = V / 256 + 64
    one = unit * (5 * mean + 4 + adds + 4 * log_sum + 1)
    entropy = unit * (5 * square + (8 + 4 + 2 * adds + 2) * mean + 2 * mean * (5 * mean + 4)) + one + \
        unit * (log_sum + mean)
    return one, 3 * unit, entropy
