"""A mixture of experts in 64 bits on the CPU, token by token, and how far a
computation in FP32 sums may be from it."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # torch.finfo(t).eps / 2


def route(x, router, k, bias=None, counts=None):
    """(chosen (B, T, k), gates (B, T, k) in 64 bits): the k experts of the
    largest x . router^T + bias, equal ones the lowest, a NaN the largest, one at
    -inf or whose bias is -inf never; the softmax of their logits.  -1 and 0 where
    none is chosen."""
    B, T, _ = x.shape
    chosen = torch.full((B, T, k), -1, dtype=torch.int32)
    gates = torch.zeros(B, T, k, dtype=torch.float64)
    logits = torch.einsum("btd,ed->bte", x.double(), router.double())
    value = logits if bias is None else torch.where(bias == -math.inf, -math.inf, logits + bias.double())
    for b in range(B):
        for t in range(T if counts is None else min(T, int(counts[b]))):
            row = value[b, t].tolist()
            order = sorted((e for e, v in enumerate(row) if v != -math.inf),
                           key=lambda e: (-math.inf if row[e] != row[e] else -row[e], row[e] == row[e], e))[:k]
            if order:
                chosen[b, t, :len(order)] = torch.tensor(order, dtype=torch.int32)
                gates[b, t, :len(order)] = torch.softmax(logits[b, t, order], -1)
    return chosen, gates


def feed_forward(x, gate_up, down, chosen, gates):
    """(y, bound): the gated sum of the chosen experts' SwiGLU blocks, (B, T, D)
    in 64 bits, and a bound on the error of a computation that sums in FP32 in
    any order (n terms: n 2^-24 of the sum of their magnitudes), rounds
    silu(g) u, gated or not, once to x's dtype and the result once; the
    exponential and the quotient take 8 steps of 2^-24 of silu."""
    B, T, D = x.shape
    E, F2, _ = gate_up.shape
    F, step, unit = F2 // 2, HALF_STEP[x.dtype], 2.0 ** -24
    k = chosen.shape[-1]
    y = torch.zeros(B, T, D, dtype=torch.float64)
    bound, size = torch.zeros_like(y), torch.zeros_like(y)
    for b in range(B):
        for t in range(T):
            row = x[b, t].double()
            for e, gate in zip(chosen[b, t].tolist(), gates[b, t].double()):
                if not 0 <= e < E:
                    continue
                w = gate_up[e].double()
                h, dh = w @ row, (D + 1) * unit * (w.abs() @ row.abs())
                g, u, dg, du = h[:F], h[F:], dh[:F], dh[F:]
                silu = g * torch.sigmoid(g)
                act = silu * u
                # silu's slope lies within -0.1 .. 1.1
                dact = 1.1 * dg * (u.abs() + du) + silu.abs() * du + (8 * unit + step) * act.abs()
                dact = dact * (1 + step + 8 * unit)
                v = down[e].double()
                term, ahead = v @ act, v.abs() @ act.abs()
                y[b, t] += gate * term
                size[b, t] += gate.abs() * ahead
                bound[b, t] += gate.abs() * (v.abs() @ dact + (F + 4 + k) * unit * (ahead + v.abs() @ dact))
    return y, bound + step * (y.abs() + bound)
