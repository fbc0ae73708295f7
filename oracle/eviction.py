"""The attention weight that cached rows receive and the rows a bounded cache
keeps, in plain loops and 64 bits: the definition the GPU forms are checked
against (no counterpart in the reference, whose cache keeps every entry)."""

import torch


def log_sum_exp(q, k, positions, scale):
    """Each query head's log-sum-exp (B, T, H) float64 over the rows it sees."""
    scores = torch.einsum("bthc,bnc->bthn", q.double(), k.double()) * scale
    unseen = torch.arange(k.shape[1]) > positions[..., None]
    return scores.masked_fill(unseen[:, :, None], float("-inf")).logsumexp(-1)


def attention_weights(q, k, positions, lse, scale, weights, counts=None, start=None):
    """New weights (B, N) float64: the old ones (zero from start[b] to the last
    counted position) plus each counted, seeing query head's exp(scale q . k -
    lse)."""
    B, T, H, _ = q.shape
    N = k.shape[1]
    out = weights.double().clone()
    for b in range(B):
        m = T if counts is None else min(max(int(counts[b]), 0), T)
        last = max([int(p) for p in positions[b, :m]], default=-1)
        last = min(last, N - 1)
        if start is not None:
            out[b, max(int(start[b]), 0):last + 1] = 0
        for t in range(m):
            p = min(int(positions[b, t]), N - 1)
            if p < 0:
                continue
            scores = q[b, t].double() @ k[b, :p + 1].double().T * scale
            out[b, :p + 1] += (scores - lse[b, t, :, None].double()).exp().sum(0)
    return out


def choose_kept(weights, lengths, keep, first, recent):
    """(kept (L, B, keep) int64, counts (B,)): weights (L, B, N)."""
    L, B, N = weights.shape
    kept = torch.full((L, B, keep), -1, dtype=torch.long)
    counts = torch.empty(B, dtype=torch.long)
    for b in range(B):
        length = min(max(int(lengths[b]), 0), N)
        counts[b] = min(length, keep)
        for i in range(L):
            rows = list(range(length))
            if length > keep:
                middle = rows[first:length - recent]
                w = [float(weights[i, b, n]) for n in middle]
                key = [float("inf") if x != x else x for x in w]
                nan = [x != x for x in w]
                best = sorted(range(len(middle)), key=lambda j: (not nan[j], -key[j], j))[:keep - first - recent]
                rows = rows[:first] + sorted(middle[j] for j in best) + rows[length - recent:]
            kept[i, b, :len(rows)] = torch.tensor(rows, dtype=torch.long)
    return kept, counts


def keep_rows(tables, kept, counts):
    """New tables (B, capacity, width): row j the old row kept[i, b, j]."""
    out = [t.clone() for t in tables]
    for i, (new, old) in enumerate(zip(out, tables)):
        for b in range(old.shape[0]):
            m = min(int(counts[b]), old.shape[1])
            rows = kept[i % kept.shape[0], b, :m]
            new[b, :m] = old[b, rows]
    return out
