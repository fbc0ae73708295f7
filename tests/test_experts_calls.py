"""Calls of the experts beside the plain ones, off the GPU: their oracle by hand
and what the entry points take and refuse."""

import math

import torch

from oracle import experts as oracle

INF, NAN = math.inf, math.nan


def test_the_oracle_leaves_out_what_a_bias_takes_out():
    x = torch.tensor([[[1.0, 2.0]]])
    router = torch.tensor([[NAN, 0.0], [INF, 0.0], [0.0, 1.0], [0.0, 2.0]])
    assert oracle.route(x, router, 2)[0].tolist() == [[[0, 1]]]
    chosen, gates = oracle.route(x, router, 3, torch.tensor([-INF, -INF, 0.0, 0.0]))
    assert chosen.tolist() == [[[3, 2, -1]]]
    assert torch.allclose(gates[0, 0], torch.tensor([1 / (1 + math.exp(-2)), 1 / (1 + math.exp(2)), 0], dtype=torch.float64))
