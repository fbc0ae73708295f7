"""oracle.experts.feed_forward for many tokens: expert by expert in matrix
products of 64 bits, on the tensors' own device."""

import torch

from oracle.experts import HALF_STEP


def feed_forward(x, gate_up, down, chosen, gates):
    """(y, bound) (rows, D) of x (rows, D), chosen and gates (rows, k), as the
    oracle gives them token by token."""
    rows, D = x.shape
    E, F2, _ = gate_up.shape
    F, step, unit, k = F2 // 2, HALF_STEP[x.dtype], 2.0 ** -24, chosen.shape[-1]
    y = torch.zeros(rows, D, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(E):
        token, slot = (chosen == e).nonzero(as_tuple=True)
        if not token.numel():
            continue
        row, gate = x[token].double(), gates[token, slot, None].double()
        w, v = gate_up[e].double().T.contiguous(), down[e].double().T.contiguous()
        h, dh = row @ w, (D + 1) * unit * (row.abs() @ w.abs())
        g, u, dg, du = h[:, :F], h[:, F:], dh[:, :F], dh[:, F:]
        silu = g * torch.sigmoid(g)
        act = silu * u
        dact = 1.1 * dg * (u.abs() + du) + silu.abs() * du + (8 * unit + step) * act.abs()
        dact = dact * (1 + step + 8 * unit)
        carried = dact @ v.abs()
        y.index_add_(0, token, gate * (act @ v))
        bound.index_add_(0, token, gate.abs() * (carried + (F + 4 + k) * unit * (act.abs() @ v.abs() + carried)))
    return y, bound + step * (y.abs() + bound)
