"""Beam search's selection and the reordering of states in plain loops and 64
bits: the definition the GPU forms are checked against (no counterpart in the
reference, whose Writer samples each row by itself)."""

import numpy as np
import torch


def log_sum_exp(x):
    """log sum exp of the float64 scores x (V,), NaN where they are none of a
    beam that can go on (a NaN, +inf, or nothing above -inf)."""
    top = x.max()
    if not np.isfinite(top):  # max of an array with a NaN is NaN
        return np.nan
    return top + np.log(np.exp(x - top).sum())


def beam_step(scores, totals, ended=None, stops=(), beams=None):
    """(totals (n, K) float64, parents, tokens, ended) by sorting every
    candidate: scores (n, W, V), totals (n, W), ended (n, W) bool."""
    n, W, V = scores.shape
    K = W if beams is None else beams
    out = [np.empty((n, K)), np.empty((n, K), np.int64), np.empty((n, K), np.int64), np.empty((n, K), bool)]
    for i in range(n):
        value = np.full((W, V), -np.inf)
        for w in range(W):
            total = float(totals[i, w])
            over = ended is not None and bool(ended[i, w])
            if not np.isfinite(total):
                continue
            if over:
                value[w, stops[0]] = total
                continue
            x = scores[i, w].double().numpy()
            level = log_sum_exp(x)
            if np.isfinite(level):
                value[w] = total + (x - level)
        order = np.argsort(-value.reshape(-1), kind="stable")[:K]
        out[0][i] = value.reshape(-1)[order]
        out[1][i], out[2][i] = order // V, order % V
        out[3][i] = [(ended is not None and bool(ended[i, w])) or v in stops for w, v in zip(out[1][i], out[2][i])]
    return tuple(torch.from_numpy(x) for x in out)


def reorder_rows(tables, parents, lengths=None):
    """New tables (n W, capacity, width): beam w of text i with the first
    lengths rows of beam parents[i, w]."""
    n, W = parents.shape
    out = [t.clone() for t in tables]
    for i in range(n):
        for w in range(W):
            source = int(parents[i, w])
            if not 0 <= source < W:
                continue
            for new, old in zip(out, tables):
                m = old.shape[1] if lengths is None else min(int(lengths[i * W + source]), old.shape[1])
                m = max(m, 0)
                new[i * W + w, :m] = old[i * W + source, :m]
    return out
