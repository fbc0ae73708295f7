"""Calls of the experts beside the plain ones, off the GPU: their oracle by hand
and what the entry points take and refuse."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from oracle import experts as oracle
from wpt_amd import kernels

INF, NAN = math.inf, math.nan


def test_the_oracle_leaves_out_what_a_bias_takes_out():
    x = torch.tensor([[[1.0, 2.0]]])
    router = torch.tensor([[NAN, 0.0], [INF, 0.0], [0.0, 1.0], [0.0, 2.0]])
    assert oracle.route(x, router, 2)[0].tolist() == [[[0, 1]]]
    chosen, gates = oracle.route(x, router, 3, torch.tensor([-INF, -INF, 0.0, 0.0]))
    assert chosen.tolist() == [[[3, 2, -1]]]
    assert torch.allclose(gates[0, 0], torch.tensor([1 / (1 + math.exp(-2)), 1 / (1 + math.exp(2)), 0], dtype=torch.float64))


def test_a_tangent_is_refused_where_it_would_be_lost():
    x, out = torch.zeros(3), torch.ones(3)
    assert kernels._forward_only(out, x, None) is out
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert kernels._forward_only(out, x, None) is out
        for call in (lambda: kernels._forward_only(out, None, x, dual), lambda: kernels._no_tangents(dual)):
            with pytest.raises(NotImplementedError):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError):  # no_grad leaves the tangents
            kernels._forward_only(out, dual)
    assert kernels._forward_only(out, dual) is out  # left behind with its level
