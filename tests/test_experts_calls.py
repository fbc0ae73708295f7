"""Calls of the experts beside the plain ones, off the GPU: their oracle by hand
and what the entry points take and refuse."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from oracle import experts as oracle
from tests import expert_sums
from wpt_amd import _lib, kernels

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


@pytest.mark.parametrize("k, D, F", [(16, 1 << 20, 32), (16, 1 << 16, 32), (8, 1 << 17, 500), (3, 1 << 20, 96), (1, 1 << 20, 8),
                                     (16, 8, 32), (8, 4096, 64)])
@pytest.mark.parametrize("dtype", [_lib.WPTV_F32, _lib.WPTV_BF16])
def test_a_round_s_terms_stay_within_512_mib(k, D, F, dtype):
    size, last = ctypes.c_size_t(), 0
    for rows in (1, 7, 8, 9, 16, 100, 512, 600, 5000, 1 << 20):
        assert _lib.lib().wptv_experts_workspace(rows, D, F, k, dtype, 0, ctypes.byref(size)) == 0
        terms = min(rows * k * D * 4, 1 << 29)
        held = min(rows, (1 << 29) // (k * D * 4)) * k * (-(-F // 32) * 32) * 4
        assert last <= size.value <= terms + held + 256
        last = size.value


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_sums_of_many_tokens_are_the_oracle_s(dtype):
    g = torch.Generator().manual_seed(0)
    x, gate_up, down = (torch.randn(*s, generator=g).to(dtype) for s in ((1, 20, 24), (5, 14, 24), (5, 24, 7)))
    chosen = torch.randint(-1, 6, (1, 20, 3), generator=g, dtype=torch.int32)
    chosen[0, 3] = torch.tensor([2, 2, 1])
    gates = torch.randn(1, 20, 3, generator=g)
    y, bound = oracle.feed_forward(x, gate_up, down, chosen, gates)
    got, limit = expert_sums.feed_forward(x[0], gate_up, down, chosen[0], gates[0])
    assert torch.allclose(got, y[0], rtol=1e-12, atol=1e-14) and torch.allclose(limit, bound[0], rtol=1e-9)
