"""Calls of the experts beside the plain ones: views of every argument, logits
and biases that are not finite."""

import math

import pytest
import torch

from oracle import experts as oracle
from wpt_amd import experts

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
BF16 = torch.bfloat16


def layer(B, T, D, E, F, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    x = normal(B, T, D).to(dtype)
    return x, normal(E, D) * D ** -0.5, (normal(E, 2 * F, D) * D ** -0.5).to(dtype), (normal(E, D, F) * F ** -0.5).to(dtype)


@pytest.mark.parametrize("rows", [3, 40, 600])
def test_given_choices_and_gates_may_both_be_views(device, rows):
    x, router, gate_up, down = (t.to(device) for t in layer(2, rows, 64, 16, 32, BF16, seed=rows))
    weights = experts.ExpertWeights(gate_up, down)
    chosen, gates = experts.route(x, router, 4)
    n = rows - 1
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (chosen, gates)]
    for rows_, c, g in ((x[:, :n], chosen[:, :n], gates[:, :n]),            # a part of the tokens
                        (x, chosen[..., 1:3], gates[..., 1:3]),             # some of the choices
                        (x, turned[0], turned[1]),
                        (x, chosen[:, :1].expand(2, rows, 4), gates[:, :1].expand(2, rows, 4))):
        held = rows_.contiguous(), c.contiguous(), g.contiguous()
        expected = experts.feed_forward(held[0], weights, held[1], held[2])
        parts = experts.feed_forward_parts(held[0], weights, held[1], held[2])
        y, bound = oracle.feed_forward(*(t.cpu() for t in (held[0][:, :2], gate_up, down, held[1][:, :2], held[2][:, :2])))
        assert bool(((expected[:, :2].cpu().double() - y).abs() <= bound).all()) and bool((y.abs().amax(-1) > 0).all())
        for _ in range(3):
            same = torch.equal(experts.feed_forward(rows_, weights, c, g), expected)
            same_parts = torch.equal(experts.feed_forward_parts(rows_, weights, c, g), parts)
            assert same and same_parts


@pytest.mark.parametrize("rows, D, E", [(1, 256, 8), (30, 64, 20), (3, 2048, 64), (200, 512, 100)])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_an_expert_taken_out_stays_out_whatever_its_logits(device, rows, D, E, value):
    print(f"route rows={rows} D={D} E={E} {value}", flush=True)
    x, router, _, _ = layer(1, rows, D, E, 8, BF16, seed=E)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(1))
    router[2, 5], bias[2] = value, -INF
    router[E - 1], bias[E - 1] = NAN, -INF
    expected = oracle.route(x, router, 4, bias)
    assert not bool(((expected[0] == 2) | (expected[0] == E - 1)).any()) and bool(expected[1].isfinite().all())
    chosen, gates = experts.route(x.to(device), router.to(device), 4, bias.to(device))
    assert torch.equal(chosen.cpu(), expected[0])
    assert bool(((gates.cpu().double() - expected[1]).abs() <= expected[1] * (2.0 ** -24 + 1e-9)).all())
